// Shared definitions of the gated delta rule (chunked forward + backward).
//
// Per value head, with state S [K, V]:
//   S <- exp(g_t) S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T;  o_t = scale S^T q_t
//
// Over a chunk of 64 tokens (gc = inclusive sum of g inside the chunk, G_ij = exp(gc_i - gc_j) for
// i >= j, S the state at the chunk's start, gC the chunk's whole sum):
//   T  = (I + A)^-1,  A_ij = beta_i G_ij k_i.k_j for i > j
//   U  = T beta (V - exp(gc) K S)                       (the u_t of the chunk)
//   O  = scale (exp(gc) Q S + (G o Q K^T) U)
//   S' = exp(gC) S + Kl^T U,                            Kl_j = exp(gC - gc_j) k_j
// With W = T beta exp(gc) K the chunk acts on its start state as an affine map,
//   S' = exp(gC) S - (Kl^T W) S + Kl^T (T beta V)  =  exp(gC) S - PM S + B,
// and its adjoint is dS = exp(gC) dS' - PM^T dS' + dB, so that everything but one [K,K] x [K,V]
// product per chunk runs in parallel over chunks.  All exponents are differences i >= j of the
// in-chunk sums (never positive for g <= 0), formed from sums held as two floats.
#pragma once
#include "common.cuh"
#include "vec.cuh"

namespace ssla {
namespace delta {

constexpr int BT = 64;            // tokens per chunk
// Rows of fp32 tiles in shared memory: 8 more than a multiple of 32 where products read pairs along
// them, 4 more where they read down the columns (no bank conflicts either way).
constexpr int LDC = BT + 8;       // [64, 64] tiles
constexpr int THREADS = 256;      // threads of the per-chunk kernels
constexpr float kMinGate = -200.f;  // exp() of less is 0 in fp32; keeps in-chunk sums finite for g = -inf

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline int64_t max_chunks(int64_t N, int64_t T) { return (T + (BT - 1) * N) / BT; }
inline int pad_k(int64_t K) { return K <= 64 ? 64 : 128; }
inline int pad_v(int64_t V) { return (int)((V + 63) / 64 * 64); }

struct Plan {
  int64_t MC;  // upper bound of chunks
  int vs;      // state columns per chain
};
Plan make_plan(int64_t N, int64_t T, int64_t HV, int64_t K, int64_t V);

// Whether the state keeps fp32 accuracy along its chain (22-bit operands, behind three planes of T for 16-bit
// tokens): for fp32 and fp16 tokens, and where a state leaves in fp32 (h0 given: its gradient may be asked
// for).  Else the chain's operands have 11 bits.  What 16-bit tokens' kernels read of the states between the
// chunks, and of their adjoints, has 16 bits either way.
inline bool exact_states(int dtype, bool h0, bool ht) { return dtype != SSLA_BF16 || h0 || ht; }
// bf16 planes of T for 16-bit tokens (delta_rule_16.cuh)
inline int t_planes(bool exact) { return exact ? 3 : 2; }

// What the forward leaves for the backward (caller's `states` buffer), states padded to KP x VP:
//   chunk_off [N+1] (device), chunk_tab [MC] {first token, rows | seq << 32}; per (chunk, value
//   head) item: tinv: T, fp32 [64,64], or for 16-bit tokens planes of it in fragment order;
//   pm: the record of pm_bytes that a step of the chain copies; s [KP,VP] = state at the chunk's
//   start, fp32, or for 16-bit tokens two bf16 planes.
struct Saved {
  int* chunk_off;
  longlong2* chunk_tab;
  float* tinv;
  unsigned char* pm;
  float* s;
};
// A chunk map's record: fp32 exp(gC) and, per 64-column panel of PM, what undoes its scale (16 bytes);
// then one or two fp16 planes [KP][KP + 8] of the scaled PM.
__host__ __device__ constexpr int pm_planes(bool exact) { return exact ? 2 : 1; }
__host__ __device__ constexpr int pm_bytes(int KP, int planes) { return 16 + 2 * planes * KP * (KP + 8); }

inline size_t saved_layout(void* base, const Plan& p, int dtype, bool exact, int64_t N, int64_t HV, int KP, int VP,
                           Saved* out) {
  char* q = (char*)base;
  const size_t items = (size_t)p.MC * HV;
  auto take = [&](size_t n) { char* r = q; q += align256(n); return (void*)r; };
  Saved s;
  s.chunk_off = (int*)take(4 * (N + 1));
  s.chunk_tab = (longlong2*)take(16 * (size_t)p.MC);
  // fp32 [64][64], or t_planes of 10 blocks of 512 bytes
  s.tinv = (float*)take((dtype == SSLA_F32 ? 4 * BT * BT : t_planes(exact) * 10 * 512) * items);
  s.pm = (unsigned char*)take(items * pm_bytes(KP, pm_planes(exact)));
  s.s = (float*)take(4 * items * KP * VP);
  if (out) *out = s;
  return (size_t)(q - (char*)base);
}

// Scratch of one call: the increments of the chunk maps (B or dB) by slices of 8 columns; for the
// backward the adjoint states (laid out as s) and, when value heads share key heads, fp32 dq and dk
// of every value head.
struct Work {
  float* inc;  // [MC*HV][VP/8][KP][8]
  float* ds;   // [MC*HV, KP, VP]
  float* dqk;  // [2, T, HV, K]
};

inline size_t work_layout(void* base, const Plan& p, int64_t T, int64_t H, int64_t HV, int64_t K, int KP, int VP,
                          bool bwd, Work* out) {
  char* q = (char*)base;
  auto take = [&](size_t n) { char* r = q; q += align256(n); return (void*)r; };
  Work w;
  const size_t states = 4 * (size_t)p.MC * HV * KP * VP;
  w.inc = (float*)take(states);
  w.ds = (float*)take(bwd ? states : 0);
  w.dqk = (float*)take(bwd && HV != H ? 8 * (size_t)T * HV * K : 0);
  if (out) *out = w;
  return (size_t)(q - (char*)base);
}
// (row, col) of an item's increments
__device__ __forceinline__ float* inc_at(float* inc, size_t item, int KP, int VP, int row, int col) {
  return inc + item * KP * VP + ((size_t)(col >> 3) * KP + row) * 8 + (col & 7);
}

// One call's tensors and sizes (device pointers), shared by the kernels.
struct Args {
  const void *q, *k, *v, *g, *beta;
  int dt_g, dt_b;
  const int64_t* cu;
  int64_t N, T, MC;
  int H, HV, R, K, V;  // R = HV / H value heads per key head
  float scale;
  bool vec_k, vec_v;  // rows of q/k, v can be copied 16 bytes at a time
};

__device__ __forceinline__ float ld_any(const void* p, int dt, size_t i) {
  if (dt == SSLA_F32) return ((const float*)p)[i];
  if (dt == SSLA_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void st_any(void* p, int dt, size_t i, float x) {
  if (dt == SSLA_F32) ((float*)p)[i] = x;
  else if (dt == SSLA_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(x);
  else ((__half*)p)[i] = __float2half_rn(x);
}

// ------------------------------------------------------------------ products of fp32 tiles
// Warp-level C += A B on mma.sync m16n8k8 TF32 with fp32 accumulators, for fp32 tokens.  Operands come
// from shared memory through functors that return a pair along the contraction, fa(row, k) =
// {A[row][k], A[row][k+1]}, fb(k, col) likewise: the order of k inside an MMA is free as long as both
// agree, so lane t takes k = 2t, 2t + 1 of every 8, one 64-bit load for tiles that are contiguous in k.
// x = hi + lo with hi the TF32 rounding, products hi hi + lo hi + hi lo, about 2^-22 relative; the
// small products have accumulators of their own, which also shortens the chain of additions that the
// tensor core truncates.  An infinity or NaN leaves lo NaN, so it is not lost.
__device__ __forceinline__ void operand(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;  // nearest, ties away
  lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

template <int MT, int NT, class FA, class FB>
__device__ __forceinline__ void warp_mma(float (&acc)[MT][NT][4], int m0, int n0, int k0, int k1, FA fa, FB fb) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
  float small[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) small[i][j][0] = small[i][j][1] = small[i][j][2] = small[i][j][3] = 0.f;
#pragma unroll 2
  for (int k = k0; k < k1; k += 8) {
    uint32_t ah[MT][4], al[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float2 x = fa(m0 + 16 * i + g, k + 2 * t), y = fa(m0 + 16 * i + g + 8, k + 2 * t);
      operand(x.x, ah[i][0], al[i][0]);
      operand(y.x, ah[i][1], al[i][1]);
      operand(x.y, ah[i][2], al[i][2]);
      operand(y.y, ah[i][3], al[i][3]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t bh[2], bl[2];
      const float2 z = fb(k + 2 * t, n0 + 8 * j + g);
      operand(z.x, bh[0], bl[0]);
      operand(z.y, bh[1], bl[1]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        mma8(acc[i][j], ah[i], bh);
        mma8(small[i][j], al[i], bh);
        mma8(small[i][j], ah[i], bl);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] += small[i][j][r];
}

// pairs along a row of a tile (contiguous), and along a column
__device__ __forceinline__ float2 pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair(const __nv_bfloat16* p) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
}
__device__ __forceinline__ float2 pair(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
template <int LD> __device__ __forceinline__ float2 column(const float* p) { return make_float2(p[0], p[LD]); }

template <int MT, int NT> __device__ __forceinline__ void zero(float (&acc)[MT][NT][4]) {
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.f;
}

// f(row, col, value0, value1) for the accumulator's pairs (row, col), (row, col + 1)
template <int MT, int NT, class F>
__device__ __forceinline__ void each_pair(float (&acc)[MT][NT][4], int m0, int n0, F f) {
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f(m0 + 16 * i + g, n0 + 8 * j + 2 * t, acc[i][j][0], acc[i][j][1]);
      f(m0 + 16 * i + g + 8, n0 + 8 * j + 2 * t, acc[i][j][2], acc[i][j][3]);
    }
}

// ------------------------------------------------------------------ scaled fp16 planes
// fp32 values as hi + lo in fp16 (22 bits) need a common power of two that brings the largest near
// 2^14.  Values down to 2^-16 of the largest then keep 22 bits; below, the low plane is subnormal and what
// is lost is absolute, 2^-38 of the largest.  (hi alone: 11 bits down to 2^-28.)  So a scale is shared only
// by values that a product adds up: a column of the state over 16 rows, 64 columns of PM.  That scale from
// the largest magnitude's bits (finite values only: an infinity must not shrink its neighbours; below
// the exponent they do not matter), and its inverse.
__device__ __forceinline__ unsigned finite_bits(float x) {
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ float plane_scale(unsigned most) {
  const unsigned e = most >> 23;  // biased exponent of the largest
  return __uint_as_float((e < 20u ? 247u : 267u - e) << 23);  // 2^(13 - exponent), at most 2^120
}
__device__ __forceinline__ float plane_unscale(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }
// plane_scale of two values at once, from the upper halves of their bits, and its inverse, as bf16 pairs
__device__ __forceinline__ uint32_t plane_scales(uint32_t most) {
  return __vminu2(0x85808580u - (most & 0x7f807f80u), 0x7b807b80u);
}
__device__ __forceinline__ uint32_t plane_unscales(uint32_t scales) { return 0x7f007f00u - scales; }
template <int N> __device__ __forceinline__ void put_half(__half* p, size_t plane, float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  *reinterpret_cast<__half2*>(p) = h;
  if (N > 1) {
    const float2 z = __half22float2(h);
    *reinterpret_cast<__half2*>(p + plane) = __floats2half2_rn(x - z.x, y - z.y);
  }
}
// w[j] of lane t of a quad <-> w[t] of lane j
__device__ __forceinline__ void quad_turn(uint32_t (&w)[4], int t) {
#pragma unroll
  for (int j = 0; j < 4; j += 2) {  // 2 x 2 blocks of neighbours
    const uint32_t x = __shfl_xor_sync(0xffffffffu, t & 1 ? w[j] : w[j + 1], 1);
    (t & 1 ? w[j] : w[j + 1]) = x;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // the blocks themselves
    const uint32_t x = __shfl_xor_sync(0xffffffffu, t & 2 ? w[j] : w[j + 2], 2);
    (t & 2 ? w[j] : w[j + 2]) = x;
  }
}
// A block's panel of PM (64 columns from c0, the accumulators of all its warps) into planes.
// red: 8 words of shared memory; ends with the block's barrier passed.
template <int KP, int NPL, int MT>
__device__ __forceinline__ void store_pm(float (&acc)[MT][4][4], int mk, int c0, int n0, unsigned* red,
                                         unsigned char* record) {
  __half* const pm = reinterpret_cast<__half*>(record + 16);
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) most = max(most, finite_bits(acc[i][j][r]));
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) most = max(most, red[w]);
  const float sc = plane_scale(most);
  if (threadIdx.x == 0) reinterpret_cast<float*>(record)[1 + c0 / 64] = plane_unscale(sc);
  // A row's 32 columns of a warp lie with the four lanes of a quad, two of every tile; turned so that
  // lane t has tile t's eight, a plane is written 16 bytes at a time (prep of the
  // 32768-token prompt of 8 heads: 350 us, with 4-byte stores 10 us more).
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t w[NPL][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = acc[i][j][2 * r] * sc, y = acc[i][j][2 * r + 1] * sc;
#pragma unroll
        for (int q = 0; q < NPL; ++q) {
          const __half2 h = __floats2half2_rn(x, y);
          const float2 z = __half22float2(h);
          w[q][j] = *reinterpret_cast<const uint32_t*>(&h);
          x -= z.x;
          y -= z.y;
        }
      }
      __half* const to = pm + (mk + 16 * i + 8 * r + g) * (KP + 8) + c0 + n0 + 8 * t;
#pragma unroll
      for (int q = 0; q < NPL; ++q) {
        quad_turn(w[q], t);
        *reinterpret_cast<uint4*>(to + (size_t)q * KP * (KP + 8)) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
      }
    }
}

// ------------------------------------------------------------------ copies into shared memory
__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// dst[64][LD] (COLS used) = rows of src; zeros behind `rows` and `cols`.  Asynchronous when vec.
template <class TI, int LD, int COLS>
__device__ __forceinline__ void load_rows(TI* dst, const TI* src, size_t stride, int rows, int cols, bool vec) {
  constexpr int E = 16 / sizeof(TI), PR = COLS / E;
  if (vec) {
    for (int i = threadIdx.x; i < BT * PR; i += THREADS) {
      const int r = i / PR, c = (i - r * PR) * E;
      if (r < rows && c < cols) cp16(dst + r * LD + c, src + r * stride + c);
      else *reinterpret_cast<uint4*>(dst + r * LD + c) = make_uint4(0, 0, 0, 0);
    }
  } else {
    for (int i = threadIdx.x; i < BT * COLS; i += THREADS) {
      const int r = i / COLS, c = i - r * COLS;
      TI x = TI(0.f);
      if (r < rows && c < cols) x = src[r * stride + c];
      dst[r * LD + c] = x;
    }
  }
}

// dst[ROWS][LD] = COLS columns of the fp32 matrix src (row length `stride`), 16-byte copies
template <int LD, int ROWS, int COLS>
__device__ __forceinline__ void load_f32(float* dst, const float* src, int stride) {
  constexpr int PR = COLS / 4;
  for (int i = threadIdx.x; i < ROWS * PR; i += THREADS) {
    const int r = i / PR, c = (i - r * PR) * 4;
    cp16(dst + r * LD + c, src + (size_t)r * stride + c);
  }
}

// ------------------------------------------------------------------ gates of one chunk
struct Gates {
  float hi[BT], lo[BT];  // in-chunk sums gc (two floats)
  float beta[BT];
  float start[BT];       // exp(gc)
  float left[BT];        // exp(gC - gc)
  float whole;           // exp(gC)
};

// Two entries of a gate array, 0 behind the end: every load leaves before the first is used.
__device__ __forceinline__ uint32_t gate_raw(const void* p, int dt, size_t i, bool in) {
  uint32_t x = 0;
  if (in && dt == SSLA_F32) x = __ldg((const uint32_t*)p + i);
  if (in && dt != SSLA_F32) x = __ldg((const unsigned short*)p + i);
  return x;
}
__device__ __forceinline__ float gate_value(uint32_t x, int dt) {
  if (dt == SSLA_F32) return __uint_as_float(x);
  if (dt == SSLA_BF16) return __uint_as_float(x << 16);
  return __half2float(__ushort_as_half((unsigned short)x));
}

// One warp.  g below kMinGate counts as kMinGate (both decay to 0), NaN stays.
__device__ __forceinline__ void load_gates(Gates& s, const Args& a, int64_t t0, int rows, int hv) {
  const int lane = threadIdx.x & 31;
  uint32_t raw[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const size_t at = (size_t)(t0 + 2 * lane + i) * a.HV + hv;
    const bool in = 2 * lane + i < rows;
    raw[i][0] = gate_raw(a.g, a.dt_g, at, in);
    raw[i][1] = gate_raw(a.beta, a.dt_b, at, in);
  }
  double x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float g = gate_value(raw[i][0], a.dt_g);
    g = g < kMinGate ? kMinGate : g;
    s.beta[2 * lane + i] = gate_value(raw[i][1], a.dt_b);
    x[i] = g;
  }
  double sum = x[0] + x[1];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  const double all = __shfl_sync(0xffffffffu, sum, 31);
  const double c[2] = {sum - x[1], sum};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 2 * lane + i;
    s.hi[r] = (float)c[i];
    s.lo[r] = (float)(c[i] - (double)s.hi[r]);
    const float e = expf(s.hi[r]);
    s.start[r] = fmaf(e, s.lo[r], e);
    s.left[r] = expf((float)(all - c[i]));
  }
  if (lane == 0) s.whole = expf((float)all);
}

// acc(i, j) *= exp(gc_i - gc_j) where i >= j (STRICT: i > j), 0 elsewhere, in place: with the stores
// of the results between them, every read of a gate would wait for its own latency.  FAST takes the
// exponential from the special-function unit (about 2^-22, for results that leave in 16 bits).
template <bool STRICT, bool FAST, int NT>
__device__ __forceinline__ void fade_scores(float (&acc)[1][NT][4], const Gates& s, int m0, int n0) {
  const int lane = threadIdx.x & 31, i0 = m0 + (lane >> 2), j0 = n0 + 2 * (lane & 3);
  const float hi[2] = {s.hi[i0], s.hi[i0 + 8]}, lo[2] = {s.lo[i0], s.lo[i0 + 8]};
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const float2 h = *reinterpret_cast<const float2*>(s.hi + j0 + 8 * t), l = *reinterpret_cast<const float2*>(s.lo + j0 + 8 * t);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + (r >> 1) * 8, j = j0 + 8 * t + (r & 1);
      const float x = (hi[r >> 1] - (r & 1 ? h.y : h.x)) + (lo[r >> 1] - (r & 1 ? l.y : l.x));
      float e;
      if (FAST) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(1.4426950408889634f * x));
      else e = expf(x);
      acc[0][t][r] = (STRICT ? i > j : i >= j) ? acc[0][t][r] * e : 0.f;
    }
  }
}

// out[i] = f acc(i, i) for the diagonal entries that a warp's accumulator holds
template <int NT>
__device__ __forceinline__ void diagonal(const float (&acc)[1][NT][4], float f, float* out, int m0, int n0) {
  const int lane = threadIdx.x & 31, i0 = m0 + (lane >> 2), j0 = n0 + 2 * (lane & 3);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + (r >> 1) * 8;
      if (i == j0 + 8 * t + (r & 1)) out[i] = f * acc[0][t][r];
    }
}

// One warp: dg of rows 2 lane, 2 lane + 1 of a chunk = sum of rc over this and the later rows + sum of
// left over the earlier ones + end.
__device__ __forceinline__ void gate_sums(const float (&rc)[2], const float (&left)[2], float end, float (&dg)[2]) {
  const int lane = threadIdx.x & 31;
  float suf = rc[0] + rc[1], pre = left[0] + left[1];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const float x = __shfl_down_sync(0xffffffffu, suf, m), y = __shfl_up_sync(0xffffffffu, pre, m);
    if (lane + m < 32) suf += x;
    if (lane >= m) pre += y;
  }
  suf = __shfl_down_sync(0xffffffffu, suf, 1);
  pre = __shfl_up_sync(0xffffffffu, pre, 1);
  if (lane == 31) suf = 0.f;
  if (lane == 0) pre = 0.f;
  const float last = rc[1] + suf;
  dg[0] = (rc[0] + last) + pre + end;
  dg[1] = last + (left[0] + pre) + end;
}

__device__ __forceinline__ bool locate(const longlong2* tab, int64_t MC, int64_t chunk, int64_t& t0, int& rows) {
  if (chunk >= MC) return false;
  const longlong2 e = tab[chunk];
  t0 = e.x;
  rows = (int)(e.y & 0xffffffff);
  return e.y >= 0;
}

// Rows of [T, n] outside every sequence become 0 (all CTAs share the work).
template <class TO>
__device__ __forceinline__ void zero_uncovered(TO* out, const Args& a, int64_t n) {
  int64_t b = a.cu[0], e = a.cu[a.N];
  b = b < 0 ? 0 : (b > a.T ? a.T : b);
  e = e < b ? b : (e > a.T ? a.T : e);
  const int64_t head = b * n, total = head + (a.T - e) * n;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x)
    out[i < head ? i : e * n + (i - head)] = TO(0.f);
}

struct Grads {
  const void* dout;
  void *dq, *dk, *dv, *dg, *dbeta;
  float* dqk;  // [2, T, HV, K] instead of dq, dk where value heads share key heads; else null
};
template <class TI>
__device__ __forceinline__ void zero_gradients(const Args& a, TI* dq, TI* dk, TI* dv, void* dg, void* dbeta, float* dqk) {
  if (dqk) {
    zero_uncovered(dqk, a, (int64_t)a.HV * a.K);
    zero_uncovered(dqk + (size_t)a.T * a.HV * a.K, a, (int64_t)a.HV * a.K);
  } else {
    zero_uncovered(dq, a, (int64_t)a.H * a.K);
    zero_uncovered(dk, a, (int64_t)a.H * a.K);
  }
  zero_uncovered(dv, a, (int64_t)a.HV * a.V);
  if (a.dt_g == SSLA_F32) zero_uncovered((float*)dg, a, a.HV);
  else zero_uncovered((__half*)dg, a, a.HV);  // 0 has the same bits in both 16-bit types
  if (a.dt_b == SSLA_F32) zero_uncovered((float*)dbeta, a, a.HV);
  else zero_uncovered((__half*)dbeta, a, a.HV);
}

// delta_rule.cu
int check_args(const char* name, int dtype, int dtype_g, int dtype_b, int64_t N, int64_t T, int64_t H, int64_t HV,
               int64_t K, int64_t V);
Args make_args(const void* q, const void* k, const void* v, const void* g, const void* beta, int dtype, int dtype_g,
               int dtype_b, const int64_t* cu, int64_t N, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V,
               float scale);
// The affine chunk maps along every sequence, from their increments w.inc: forward S' = decay S - PM S + B
// (s: start states), reverse the adjoint with PM^T (s: adjoint of every chunk's end state).  exact:
// products at fp32 accuracy; planes: s in two bf16 planes instead of fp32.
int run_chain(const Plan& p, const Saved& sv, const Work& w, float* s, const float* init, float* last, int64_t N,
              int HV, int K, int V, bool reverse, bool exact, bool planes, cudaStream_t st);
// delta_rule_16.cu, delta_rule_16_bwd.cu: the per-chunk kernels of 16-bit tokens
int prep16(int dtype, const Args& a, const Saved& sv, int KP, int VP, bool exact, float* inc, int64_t items,
           cudaStream_t st);
int output16(int dtype, const Args& a, const Saved& sv, int KP, int VP, bool exact, void* o, int64_t items,
             cudaStream_t st);
int adjoint16(int dtype, const Args& a, const Saved& sv, int KP, int VP, int planes, const void* dout, float* inc,
              int64_t items, cudaStream_t st);
int backward16(int dtype, const Args& a, const Saved& sv, int KP, int VP, int planes, const void* ds, const Grads& g,
               int64_t items, cudaStream_t st);

}  // namespace delta
}  // namespace ssla
