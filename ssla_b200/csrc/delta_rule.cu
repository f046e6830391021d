// Chunked gated delta rule, forward (delta_rule.cuh has the formulas).
//   tables      chunk list of the packed sequences (pack_tables.cu; device only, no host read)
//   prep        per (chunk, value head): T, PM = Kl^T W, B = Kl^T T beta V, exp(gC)
//   chain       S' = exp(gC) S - PM S + B along every sequence: the one sequential part
//   output      per (chunk, value head): O from the start state
// The prep and output kernels here are those of fp32 tokens (split TF32 products); the chain serves
// every type.
#include "delta_rule_16.cuh"
#include "delta_rule_inverse.cuh"
#include "pack_tables.cuh"
#include "tc_util.cuh"

namespace ssla {
namespace delta {
namespace {

// ------------------------------------------------------------------ prep
using TI = float;  // 16-bit tokens: delta_rule_16.cu

template <int KP> struct PrepSmem {
  static constexpr int LDK = KP + 8, LDV = 72;
  TI k[BT * LDK];
  TI v[BT * LDV];
  float a[BT * LDC];
  float t[BT * LDC];
  float y[BT * 68];
  float col[BT];
  unsigned red[THREADS / 32];
  Gates gates;
};

template <int KP>
__global__ void __launch_bounds__(THREADS, 2) prep_kernel(Args a, const longlong2* __restrict__ tab, int VP,
                                                          float* __restrict__ tinv, unsigned char* __restrict__ pm,
                                                          float* __restrict__ inc) {
  griddep_launch_dependents();
  griddep_wait();
  using S = PrepSmem<KP>;
  constexpr int LDK = S::LDK, LDV = S::LDV;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
  unsigned char* const record = pm + item * pm_bytes(KP, 2);
  const int warp = threadIdx.x >> 5;
  load_rows<TI, LDK, KP>(s.k, (const TI*)a.k + ((size_t)t0 * a.H + h) * a.K, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  auto load_v = [&](int v0) {
    load_rows<TI, LDV, 64>(s.v, (const TI*)a.v + ((size_t)t0 * a.HV + hv) * a.V + v0, (size_t)a.HV * a.V, rows,
                           a.V - v0, a.vec_v);
  };
  load_v(0);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  cp_wait<0>();
  __syncthreads();
  if (threadIdx.x == 0) *reinterpret_cast<float*>(record) = s.gates.whole;
  const TI* sk = s.k;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  {
    float acc[1][4][4];
    zero(acc);
    if (n0 <= m0)
      warp_mma(acc, m0, n0, 0, KP, [&](int m, int k) { return pair(sk + m * LDK + k); },
                         [&](int k, int n) { return pair(sk + n * LDK + k); });
    fade_scores<true, false>(acc, s.gates, m0, n0);
    const int i0 = m0 + ((threadIdx.x & 31) >> 2);
    const float b0 = s.gates.beta[i0], b1 = s.gates.beta[i0 + 8];
    each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
      const float b = i == i0 ? b0 : b1;
      *reinterpret_cast<float2*>(s.a + i * LDC + j) = make_float2(b * x, b * y);
    });
  }
  __syncthreads();
  unit_lower_inverse(s.a, s.t, s.y);
  for (int i = threadIdx.x; i < BT * 16; i += THREADS) {
    const int r = i >> 4, c = (i & 15) * 4;
    *reinterpret_cast<float4*>(tinv + item * (BT * BT) + r * BT + c) = *reinterpret_cast<float4*>(s.t + r * LDC + c);
  }
  // panels of 64 columns of [W | T beta V], each followed by its product with Kl^T
  const int panels = KP / 64 + VP / 64;
  for (int p = 0; p < panels; ++p) {
    const bool w = p < KP / 64;
    const int c0 = (w ? p : p - KP / 64) * 64;
    __syncthreads();  // the previous panel's readers of col, v and y are done
    if (threadIdx.x < BT) s.col[threadIdx.x] = s.gates.beta[threadIdx.x] * (w ? s.gates.start[threadIdx.x] : 1.f);
    if (!w && c0 > 0) {
      load_v(c0);
      cp_commit();
      cp_wait<0>();
    }
    __syncthreads();
    {
      float acc[1][4][4];
      zero(acc);
      auto fa = [&](int i, int j) {
        const float2 x = pair(s.t + i * LDC + j), c = pair(s.col + j);
        return make_float2(x.x * c.x, x.y * c.y);
      };
      if (w)
        warp_mma(acc, m0, n0, 0, m0 + 16, fa, [&](int j, int n) { return column<LDK>(sk + j * LDK + c0 + n); });
      else
        warp_mma(acc, m0, n0, 0, m0 + 16, fa, [&](int j, int n) { return column<LDV>(s.v + j * LDV + n); });
      each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
        const float l = s.gates.left[i];
        *reinterpret_cast<float2*>(s.y + i * 68 + j) = make_float2(x * l, y * l);
      });
    }
    __syncthreads();
    {
      constexpr int MT = KP / 64;
      float acc[MT][4][4];
      zero(acc);
      const int mk = (warp >> 1) * 16 * MT;
      warp_mma(acc, mk, n0, 0, BT, [&](int m, int j) { return column<LDK>(sk + j * LDK + m); },
                           [&](int j, int n) { return column<68>(s.y + j * 68 + n); });
      if (w)
        store_pm<KP, 2>(acc, mk, c0, n0, s.red, record);
      else
        each_pair(acc, mk, n0, [&](int m, int n, float x, float y) {
          *reinterpret_cast<float2*>(inc_at(inc, item, KP, VP, m, c0 + n)) = make_float2(x, y);
        });
    }
  }
}

// ------------------------------------------------------------------ chain
// One CTA carries VS columns of one state along its sequence's chunks; every warp owns 16 of the KP
// rows in the accumulator layout (fp32).  The one product of a step, PM S, runs on fp16 planes (NP =
// 2: hi + lo, 22 bits, three MMAs; NP = 1: 11 bits, for states whose only readers are bf16 outputs):
// prep leaves PM in planes scaled by a power of two per 64 columns, and every warp scales each column of
// its 16 rows of S by one of its own before it shares them, undone when the MMA over those 16 rows of
// the contraction is added.  Value columns never meet, so none may set another's scale: with one scale for
// a warp's columns, a column 1e-8 times its neighbour had lost half its bits, and which columns share it
// went with the number of chains.  A step streams the chunk's record and its slice of B through a ring
// of bulk copies (a warp of its own issues them; the memory has the layout of shared memory), and has one
// barrier.  A wait that gives up makes the rest of the chain NaN.
// What bounds it: the dependent chain of a step (barrier, MMAs, rescaling), 0.66 us for 64 x 64; for
// 128 x 128 at fp32 accuracy the 74 KB a step from L2 too, 1.03 us with 8 columns on 128 SMs.  The scales by
// column are 0.06 and 0.09 us of that (three dependent shuffles; reductions of the warp under four masks
// instead: 1.35 us).  Before they came, at 0.95 us and 92 us for 112 chains of 32 columns (105 us now):
// two CTAs that share a state over distributed shared memory halve the bytes, but the cluster barrier took a
// step to 1.7 us; two buffers instead of three, 2.0 us; two blocks per SM for 32 columns, with B in
// registers, 106 us; states leaving in 4-byte instead of 16-byte pieces, 117 us.
template <int KP, int VS, int NP> struct ChainSmem {
  static constexpr int LDP = KP + 8, LDS = VS == 8 ? 8 : VS + 8;  // ldmatrix without conflicts
  static constexpr int PM = pm_bytes(KP, NP), B = 4 * KP * VS, STAGE = PM + B;  // bytes
  // two buffers of the state's planes and of what undoes their scales: bf16 [KP / 16][4 lanes][tile][2 columns]
  static constexpr int S = 2 * NP * KP * LDS, UN = 2 * (KP / 16) * VS, STATE = 2 * (S + UN), MOST = 227 * 1024 - 1024;
  static constexpr int fit = (MOST - STATE - 64) / STAGE, stages = fit > 4 ? 4 : fit, bytes = STATE + 64 + stages * STAGE;
  static_assert(stages >= 2 && STATE % 32 == 0 && STAGE % 16 == 0, "a step is loaded while another runs");
};

struct ChainArgs {
  const unsigned char* pm;  // [item] records
  const float* inc;         // [item][VP / 8][KP][8]
  float* s;          // start (reverse: end) state of every chunk [item][KP][VP], in two bf16 planes if planes
  const int* off;    // chunks of sequence n: off[n] .. off[n + 1] - 1; item = chunk * HV + head
  const float* init; // [N * HV][K][V] or null
  float* last;       // likewise
  bool reverse, planes;
  int HV, K, V, VP, slices;
};

// 16-byte aligned addresses, bytes a multiple of 16; completes on the mbarrier
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   h16::smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(h16::smem_u32(mbar))
               : "memory");
}

__device__ __forceinline__ void mma16h(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int KP, int VS, bool TRANS, int NP>
__global__ void __launch_bounds__(KP * 2 + 32) chain_kernel(ChainArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  using M = ChainSmem<KP, VS, NP>;
  constexpr int NT = VS / 8, LDP = M::LDP, LDS = M::LDS, ST = M::stages, NB = KP / 16;
  extern __shared__ __align__(16) unsigned char raw[];
  uint64_t* const full = reinterpret_cast<uint64_t*>(raw + M::STATE);
  unsigned char* const ring = raw + M::STATE + 64;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, m0 = warp * 16;
  const unsigned lh = blockIdx.x / (unsigned)a.slices;
  const int c0 = (int)(blockIdx.x - lh * a.slices) * VS;
  const int list = (int)(lh / (unsigned)a.HV), hv = (int)(lh - (unsigned)list * a.HV);
  const int first = a.off[list], count = a.off[list + 1] - first;
  auto at = [&](int i) { return (size_t)(first + (a.reverse ? count - 1 - i : i)) * a.HV + hv; };
  auto load = [&](int i) {  // one thread
    const size_t it = at(i);
    unsigned char* dst = ring + (i % ST) * M::STAGE;
    tc::mbar_arrive_expect_tx(full + i % ST, M::STAGE);
    bulk_load(dst, a.pm + it * M::PM, M::PM, full + i % ST);
    bulk_load(dst + M::PM, a.inc + it * KP * a.VP + (size_t)c0 * KP, M::B, full + i % ST);
  };
  const bool producer = warp == KP / 16;
  if (producer && lane == 0) {
    for (int i = 0; i < ST; ++i) tc::mbar_init(full + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < ST - 1 && i < count; ++i) load(i);
  }
  __syncthreads();
  bool good = true;
  if (producer) {
    int late = 0;  // copies under way when a wait gave up
    for (int i = 0; i < count; ++i) {
      if (good && !tc::mbar_wait(full + i % ST, (i / ST) & 1, 1u << 20)) {
        good = false;
        late = i;
      }
      __syncthreads();
      if (lane == 0 && good && i + ST - 1 < count) load(i + ST - 1);
    }
    if (!good)  // let them end, within limits, before the block's memory goes
      for (int i = late; i < late + ST - 1 && i < count; ++i) tc::mbar_wait(full + i % ST, (i / ST) & 1, 1u << 20);
    return;
  }
  float S[1][NT][4];
  each_pair(S, m0, 0, [&](int r, int c, float& x, float& y) {
    x = y = 0.f;
    const int cc = c0 + c;
    if (a.init && r < a.K) {
      const float* p = a.init + ((size_t)lh * a.K + r) * a.V + cc;
      if (cc < a.V) x = p[0];
      if (cc + 1 < a.V) y = p[1];
    }
  });
  // lane addresses of ldmatrix: the map's rows (its transpose: columns), the state's rows
  const uint32_t a_at = TRANS ? ((lane & 7) + (lane >> 4) * 8) * LDP + ((lane >> 3) & 1) * 8 + m0
                              : (m0 + (lane & 15)) * LDP + (lane >> 4) * 8;
  const uint32_t b_at = VS == 8 ? (lane & 15) * LDS + (NP > 1 ? (lane >> 4) * (KP * LDS) : 0)
                                : ((lane & 7) + ((lane >> 3) & 1) * 8) * LDS + (lane >> 4) * 8;
  for (int i = 0; i < count; ++i) {
    const size_t it = at(i);
    __half* sc = reinterpret_cast<__half*>(raw + (i & 1) * (M::STATE / 2));
    uint32_t* un = reinterpret_cast<uint32_t*>(raw + (i & 1) * (M::STATE / 2) + M::S);
    // largest exponents of a lane's two columns of each tile, in the halves of a word, over the 16 rows
    unsigned most[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      most[j] = __byte_perm(max(finite_bits(S[0][j][0]), finite_bits(S[0][j][2])),
                            max(finite_bits(S[0][j][1]), finite_bits(S[0][j][3])), 0x7632);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1)
#pragma unroll
      for (int j = 0; j < NT; ++j) most[j] = __vmaxu2(most[j], __shfl_xor_sync(0xffffffffu, most[j], d));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t scales = plane_scales(most[j]);
      const float x = __uint_as_float(scales << 16), y = __uint_as_float(scales & 0xffff0000u);
      if (g == 0) un[(warp * 4 + t) * NT + j] = plane_unscales(scales);
#pragma unroll
      for (int r = 0; r < 2; ++r)
        put_half<NP>(sc + (m0 + g + 8 * r) * LDS + 8 * j + 2 * t, KP * LDS, S[0][j][2 * r] * x, S[0][j][2 * r + 1] * y);
    }
    good = good && tc::mbar_wait(full + i % ST, (i / ST) & 1, 1u << 20);
    __syncthreads();  // the state is there, step i - 1 is read
    const unsigned char* stage = ring + (i % ST) * M::STAGE;
    const float* ps = reinterpret_cast<const float*>(stage) + 1;
    const float d = good ? ps[-1] : __int_as_float(0x7fffffff);
    const uint32_t pa = h16::smem_u32(stage + 16) + 2 * a_at, pb = h16::smem_u32(sc) + 2 * b_at;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    // products of 16 rows of the contraction; of a single column tile all of them stay open while the
    // state is stored
    float parts[NT == 1 ? NB : 1][NT][4];
    float u[NT == 1 ? NB : 1][2 * NT];  // what undoes the scales of a lane's columns, times PM's
    auto undo = [&](int kb) {
      const float f = TRANS ? 1.f : ps[kb / 4];
      const uint32_t* p = un + (kb * 4 + t) * NT;
      uint32_t w[NT];
      if constexpr (NT == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      } else if constexpr (NT == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x; w[1] = x.y;
      } else {
        w[0] = *p;
      }
      float(&v)[2 * NT] = u[NT == 1 ? kb : 0];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        v[2 * j] = f * __uint_as_float(w[j] << 16);
        v[2 * j + 1] = f * __uint_as_float(w[j] & 0xffff0000u);
      }
    };
    if (NT == 1)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) undo(kb);
    auto join = [&](int kb) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[j][r] = fmaf(u[NT == 1 ? kb : 0][2 * j + (r & 1)], parts[NT == 1 ? kb : 0][j][r], acc[j][r]);
    };
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      uint32_t fa[NP][4];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint32_t q = pa + 2 * (p * KP * LDP + (TRANS ? kb * 16 * LDP : kb * 16));
        if (TRANS) h16::ldsm4t(fa[p], q);
        else h16::ldsm4(fa[p], q);
      }
      uint32_t fb[NP][NT][2];
      if (VS == 8) {  // both planes of the one column tile at once (one plane: the upper half is unused)
        uint32_t r[4];
        h16::ldsm4t(r, pb + 2 * kb * 16 * LDS);
        fb[0][0][0] = r[0];
        fb[0][0][1] = r[1];
        fb[NP - 1][0][0] = r[NP > 1 ? 2 : 0];
        fb[NP - 1][0][1] = r[NP > 1 ? 3 : 1];
      } else {
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int j = 0; j < NT; j += 2) {
            uint32_t r[4];
            h16::ldsm4t(r, pb + 2 * (p * KP * LDS + kb * 16 * LDS + 8 * j));
            fb[p][j][0] = r[0];
            fb[p][j][1] = r[1];
            fb[p][j + (NT > 1)][0] = r[2];
            fb[p][j + (NT > 1)][1] = r[3];
          }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float(&part)[4] = parts[NT == 1 ? kb : 0][j];
        part[0] = part[1] = part[2] = part[3] = 0.f;
        if (NP > 1) {
          mma16h(part, fa[NP - 1], fb[0][j][0], fb[0][j][1]);
          mma16h(part, fa[0], fb[NP - 1][j][0], fb[NP - 1][j][1]);
        }
        mma16h(part, fa[0], fb[0][j][0], fb[0][j][1]);
      }
      if (NT > 1) {
        undo(kb);
        join(kb);
      }
    }
    if (a.s && a.planes) {
      // piece q: plane q / 2 NT, row g + 8 (q / NT % 2), tile q % NT; a quad turns four of them, so that
      // lane t writes 16 bytes of piece 4 u + t
      uint32_t w[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = S[0][j][2 * r], y = S[0][j][2 * r + 1];
          const int hi = r * NT + j, lo = hi + 2 * NT;
          w[hi / 4][hi % 4] = h16::pack(x, y);
          h16::rest(w[hi / 4][hi % 4], x, y);
          w[lo / 4][lo % 4] = h16::pack(x, y);
        }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        quad_turn(w[u], t);
        const int q = 4 * u + t, row = m0 + g + 8 * (q / NT % 2);
        h16::bf* const to = (h16::bf*)a.s + ((2 * it + q / (2 * NT)) * KP + row) * a.VP + c0 + 8 * (q % NT);
        *reinterpret_cast<uint4*>(to) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
      }
    } else if (a.s) {
      each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
        *reinterpret_cast<float2*>(a.s + (it * KP + r) * a.VP + c0 + c) = make_float2(x, y);
      });
    }
    if (NT == 1)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) join(kb);
    const float* bc = reinterpret_cast<const float*>(stage + M::PM);
    const float f = TRANS ? ps[m0 / 64] : 1.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 b = pair(bc + (j * KP + m0 + g + 8 * r) * 8 + 2 * t);
        float &x = S[0][j][2 * r], &y = S[0][j][2 * r + 1];
        x = fmaf(d, x, b.x - f * acc[j][2 * r]);
        y = fmaf(d, y, b.y - f * acc[j][2 * r + 1]);
      }
  }
  if (a.last)
    each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
      const int cc = c0 + c;
      if (r < a.K) {
        float* p = a.last + ((size_t)lh * a.K + r) * a.V + cc;
        if (cc < a.V) p[0] = x;
        if (cc + 1 < a.V) p[1] = y;
      }
    });
}

template <int KP, int VS, bool TRANS, int NP> int launch_chain(const ChainArgs& a, int64_t N, cudaStream_t st) {
  constexpr int smem = ChainSmem<KP, VS, NP>::bytes;
  allow_smem<chain_kernel<KP, VS, TRANS, NP>>((int)smem);
  const int64_t grid = N * a.HV * a.slices;
  if (grid == 0) return SSLA_OK;
  // after its predecessor, not into its tail: there the blocks would pile up on the SMs that are free
  // first (8 x 2048 tokens, 4 heads of 64: 30 us instead of 19)
  chain_kernel<KP, VS, TRANS, NP><<<(unsigned)grid, KP * 2 + 32, smem, st>>>(a);
  SSLA_CHECK_LAUNCH("gated_delta_rule chain");
  return SSLA_OK;
}

template <int KP, int VS> int chain_vs(const ChainArgs& a, bool exact, int64_t N, cudaStream_t st) {
  if (exact) return a.reverse ? launch_chain<KP, VS, true, 2>(a, N, st) : launch_chain<KP, VS, false, 2>(a, N, st);
  return a.reverse ? launch_chain<KP, VS, true, 1>(a, N, st) : launch_chain<KP, VS, false, 1>(a, N, st);
}

template <int KP> int chain_kp(const ChainArgs& a, int vs, bool exact, int64_t N, cudaStream_t st) {
  if (vs == 8) return chain_vs<KP, 8>(a, exact, N, st);
  if (vs == 16) return chain_vs<KP, 16>(a, exact, N, st);
  return chain_vs<KP, 32>(a, exact, N, st);
}

// ------------------------------------------------------------------ output
template <int KP, int VB> struct OutSmem {
  static constexpr int LDK = KP + 8, LDV = VB + 8, LDX = VB + 4;
  TI k[BT * LDK];
  TI q[BT * LDK];
  TI v[BT * LDV];
  float p[BT * LDC];
  float t[BT * LDC];
  float s[KP * LDX];
  float x[BT * LDX];
  Gates gates;
};

template <int KP, int VB>
__device__ __forceinline__ void output_chunk(const Args& a, const longlong2* __restrict__ tab, int VP,
                                             const float* __restrict__ tinv, const float* __restrict__ states,
                                             TI* __restrict__ o) {
  using S = OutSmem<KP, VB>;
  constexpr int LDK = S::LDK, LDV = S::LDV, LDX = S::LDX, NT = VB / 16;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
  const int warp = threadIdx.x >> 5;
  const size_t qk = ((size_t)t0 * a.H + h) * a.K;
  load_rows<TI, LDK, KP>(s.k, (const TI*)a.k + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_rows<TI, LDK, KP>(s.q, (const TI*)a.q + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_f32<LDC, BT, BT>(s.t, tinv + item * (BT * BT), BT);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  const TI *sk = s.k, *sq = s.q;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * (VB / 2);
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V;
  const float* st = states + item * KP * VP;
  for (int v0 = 0; v0 < a.V; v0 += VB) {
    __syncthreads();  // readers of the previous panel are done
    load_f32<LDX, KP, VB>(s.s, st + v0, VP);
    load_rows<TI, LDV, VB>(s.v, (const TI*)a.v + vo + v0, (size_t)a.HV * a.V, rows, a.V - v0, a.vec_v);
    cp_commit();
    if (v0 == 0) {  // P = (G o Q K^T), while the first state panel is under way
      cp_wait<1>();
      __syncthreads();
      const int p0 = (warp & 1) * 32;
      float acc[1][4][4];
      zero(acc);
      if (p0 <= m0)
        warp_mma(acc, m0, p0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); },
                           [&](int k, int n) { return pair(sk + n * LDK + k); });
      fade_scores<false, false>(acc, s.gates, m0, p0);
      each_pair(acc, m0, p0, [&](int i, int j, float x, float y) {
        *reinterpret_cast<float2*>(s.p + i * LDC + j) = make_float2(x, y);
      });
    }
    cp_wait<0>();
    __syncthreads();
    float aq[1][NT][4], ak[1][NT][4];
    zero(aq);
    zero(ak);
    auto fs = [&](int k, int n) { return column<LDX>(s.s + k * LDX + n); };
    warp_mma(ak, m0, n0, 0, KP, [&](int m, int k) { return pair(sk + m * LDK + k); }, fs);
    warp_mma(aq, m0, n0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); }, fs);
    each_pair(ak, m0, n0, [&](int i, int n, float x, float y) {
      const float b = s.gates.beta[i], e = s.gates.start[i];
      *reinterpret_cast<float2*>(s.x + i * LDX + n) =
          make_float2(b * (ldf(s.v + i * LDV + n) - e * x), b * (ldf(s.v + i * LDV + n + 1) - e * y));
    });
    __syncthreads();
    zero(ak);
    auto fx = [&](int k, int n) { return column<LDX>(s.x + k * LDX + n); };
    warp_mma(ak, m0, n0, 0, m0 + 16, [&](int m, int k) { return pair(s.t + m * LDC + k); }, fx);
    __syncthreads();
    each_pair(ak, m0, n0, [&](int i, int n, float x, float y) {
      *reinterpret_cast<float2*>(s.x + i * LDX + n) = make_float2(x, y);
    });
    each_pair(aq, m0, n0, [&](int i, int, float& x, float& y) {
      x *= s.gates.start[i];
      y *= s.gates.start[i];
    });
    __syncthreads();
    warp_mma(aq, m0, n0, 0, m0 + 16, [&](int m, int k) { return pair(s.p + m * LDC + k); }, fx);
    each_pair(aq, m0, n0, [&](int i, int n, float x, float y) {
      const int c = v0 + n;
      if (i < rows) {
        TI* p = o + vo + (size_t)i * a.HV * a.V + c;
        if (c < a.V) stf(p, x * a.scale);
        if (c + 1 < a.V) stf(p + 1, y * a.scale);
      }
    });
  }
}

template <int KP, int VB>
__global__ void __launch_bounds__(THREADS, 2) output_kernel(Args a, const longlong2* __restrict__ tab, int VP,
                                                            const float* __restrict__ tinv,
                                                            const float* __restrict__ states, TI* __restrict__ o) {
  griddep_launch_dependents();
  griddep_wait();
  output_chunk<KP, VB>(a, tab, VP, tinv, states, o);
  zero_uncovered(o, a, (int64_t)a.HV * a.V);
}

template <int KP>
int prep32(const Args& a, const Saved& sv, int VP, float* inc, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(PrepSmem<KP>);
  allow_smem<prep_kernel<KP>>((int)smem);
  launch_pdl(prep_kernel<KP>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, sv.tinv, sv.pm, inc);
  SSLA_CHECK_LAUNCH("gated_delta_rule prep");
  return SSLA_OK;
}

template <int KP>
int output32(const Args& a, const Saved& sv, int VP, void* o, int64_t items, cudaStream_t st) {
  constexpr int VB = KP == 64 ? 64 : 32;
  const size_t smem = sizeof(OutSmem<KP, VB>);
  allow_smem<output_kernel<KP, VB>>((int)smem);
  launch_pdl(output_kernel<KP, VB>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, sv.tinv, sv.s, (TI*)o);
  SSLA_CHECK_LAUNCH("gated_delta_rule output");
  return SSLA_OK;
}

}  // namespace

Plan make_plan(int64_t N, int64_t T, int64_t HV, int64_t K, int64_t V) {
  Plan p;
  p.MC = max_chunks(N, T);
  const int VP = pad_v(V);
  // Columns of a chain: 8 while that leaves few blocks (a step is its own latency: 512 steps of 128 x
  // 128 take 0.53 ms with 8 columns on 128 SMs, 0.70 ms with 16 on 64), up to 32 while at least two
  // blocks per SM remain (the map is read once per block: 112 chains of 128 x 128 take 213 us with 8
  // columns, 130 us with 16, 105 us with 32).
  p.vs = 8;
  while (p.vs < 32 && N * HV * (VP / (2 * p.vs)) >= 2 * kNumSMs) p.vs *= 2;
  return p;
}

int check_args(const char* name, int dtype, int dtype_g, int dtype_b, int64_t N, int64_t T, int64_t H, int64_t HV,
               int64_t K, int64_t V) {
  SSLA_CHECK_ARG(dtype_ok(dtype) && dtype_ok(dtype_g) && dtype_ok(dtype_b), "%s: bad dtype", name);
  SSLA_CHECK_ARG(N >= 0 && T >= 0 && H >= 0 && HV >= 0, "%s: negative size", name);
  SSLA_CHECK_ARG(H > 0 ? HV % H == 0 : HV == 0, "%s: %lld value heads over %lld key heads", name, (long long)HV,
                 (long long)H);
  SSLA_CHECK_ARG(K >= 1 && V >= 1 && K <= 128 && V <= 256, "%s: K=%lld V=%lld not supported (1 <= K <= 128, 1 <= V <= 256)",
                 name, (long long)K, (long long)V);
  SSLA_CHECK_ARG(N < (int64_t(1) << 31) && (max_chunks(N, T) + N) * (HV > 0 ? HV : 1) < (int64_t(1) << 25),
                 "%s: too many chunks (%lld sequences, %lld tokens, %lld heads)", name, (long long)N, (long long)T,
                 (long long)HV);
  return SSLA_OK;
}

Args make_args(const void* q, const void* k, const void* v, const void* g, const void* beta, int dtype, int dtype_g,
               int dtype_b, const int64_t* cu, int64_t N, int64_t T, int64_t H, int64_t HV, int64_t K, int64_t V,
               float scale) {
  Args a;
  a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta;
  a.dt_g = dtype_g; a.dt_b = dtype_b;
  a.cu = cu;
  a.N = N; a.T = T; a.MC = max_chunks(N, T);
  a.H = (int)H; a.HV = (int)HV; a.R = H > 0 ? (int)(HV / H) : 1;
  a.K = (int)K; a.V = (int)V;
  a.scale = scale;
  const size_t e = dtype_size(dtype);
  a.vec_k = K * e % 16 == 0 && aligned_to(q, 16) && aligned_to(k, 16);
  a.vec_v = V * e % 16 == 0 && aligned_to(v, 16);
  return a;
}

int run_chain(const Plan& p, const Saved& sv, const Work& w, float* s, const float* init, float* last, int64_t N,
              int HV, int K, int V, bool reverse, bool exact, bool planes, cudaStream_t st) {
  ChainArgs c = {};
  c.pm = sv.pm;
  c.inc = w.inc;
  c.s = s;
  c.off = sv.chunk_off;
  c.init = init;
  c.last = last;
  c.reverse = reverse;
  c.planes = planes;
  c.HV = HV;
  c.K = K;
  c.V = V;
  c.VP = pad_v(V);
  c.slices = c.VP / p.vs;
  return pad_k(K) == 64 ? chain_kp<64>(c, p.vs, exact, N, st) : chain_kp<128>(c, p.vs, exact, N, st);
}

}  // namespace delta
}  // namespace ssla

using namespace ssla;
using namespace ssla::delta;

extern "C" size_t ssla_gated_delta_rule_states_bytes(int dtype, int64_t n_seqs, int64_t T, int64_t H, int64_t HV,
                                                     int64_t K, int64_t V, int has_h0, int has_ht) {
  if (n_seqs < 0 || T < 0 || H < 0 || HV < 0 || K < 1 || V < 1) return 0;
  return saved_layout(nullptr, make_plan(n_seqs, T, HV, K, V), dtype, exact_states(dtype, has_h0, has_ht), n_seqs, HV,
                      pad_k(K), pad_v(V), nullptr);
}

extern "C" size_t ssla_gated_delta_rule_workspace_bytes(int64_t n_seqs, int64_t T, int64_t H, int64_t HV, int64_t K,
                                                        int64_t V, int backward) {
  if (n_seqs < 0 || T < 0 || H < 0 || HV < 0 || K < 1 || V < 1) return 0;
  return work_layout(nullptr, make_plan(n_seqs, T, HV, K, V), T, H, HV, K, pad_k(K), pad_v(V), backward != 0, nullptr);
}

extern "C" int ssla_chunk_gated_delta_rule_fwd(const void* q, const void* k, const void* v, const void* g,
                                               const void* beta, int dtype, int dtype_g, int dtype_beta,
                                               const int64_t* cu_seqlens, int64_t n_seqs, int64_t T, int64_t H,
                                               int64_t HV, int64_t K, int64_t V, float scale, const float* h0, void* o,
                                               float* ht, void* states, size_t states_bytes, void* workspace,
                                               size_t workspace_bytes, ssla_stream_t stream) {
  const char* name = "ssla_chunk_gated_delta_rule_fwd";
  int rc = check_args(name, dtype, dtype_g, dtype_beta, n_seqs, T, H, HV, K, V);
  if (rc) return rc;
  if (HV == 0) return SSLA_OK;
  SSLA_CHECK_ARG(cu_seqlens && states, "%s: null pointer", name);
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta), "%s: null pointer", name);
  const Plan p = make_plan(n_seqs, T, HV, K, V);
  const int KP = pad_k(K), VP = pad_v(V);
  const bool exact = exact_states(dtype, h0, ht);
  Saved sv;
  Work w;
  const size_t need = saved_layout(states, p, dtype, exact, n_seqs, HV, KP, VP, &sv);
  const size_t need_w = work_layout(workspace, p, T, H, HV, K, KP, VP, false, &w);
  if (states_bytes < need || workspace_bytes < need_w || (need_w && !workspace)) {
    set_error("%s: states of %zu bytes and workspace of %zu, %zu and %zu needed", name, states_bytes, workspace_bytes,
              need, need_w);
    return SSLA_ERR_WORKSPACE;
  }
  SSLA_CHECK_ARG(aligned_to(states, 16) && aligned_to(workspace, 16), "%s: states and workspace must be 16-byte aligned", name);
  cudaStream_t st = (cudaStream_t)stream;
  rc = launch_pack_tables(cu_seqlens, n_seqs, T, BT, p.MC, sv.chunk_off, sv.chunk_tab, st);
  if (rc) return rc;
  const Args a = make_args(q, k, v, g, beta, dtype, dtype_g, dtype_beta, cu_seqlens, n_seqs, T, H, HV, K, V, scale);
  const int64_t items = p.MC * HV, blocks = items > 0 ? items : 1;
  const bool f32 = dtype == SSLA_F32;
  if (items > 0) {
    rc = !f32      ? prep16(dtype, a, sv, KP, VP, exact, w.inc, items, st)
         : KP == 64 ? prep32<64>(a, sv, VP, w.inc, items, st)
                    : prep32<128>(a, sv, VP, w.inc, items, st);
    if (rc) return rc;
  }
  rc = run_chain(p, sv, w, sv.s, h0, ht, n_seqs, (int)HV, (int)K, (int)V, false, exact, !f32, st);
  if (rc || T == 0 || !o) return rc;
  return !f32       ? output16(dtype, a, sv, KP, VP, exact, o, blocks, st)
         : KP == 64 ? output32<64>(a, sv, VP, o, blocks, st)
                    : output32<128>(a, sv, VP, o, blocks, st);
}
