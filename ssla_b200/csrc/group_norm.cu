// Group norm with an activation over channels-last rows x [T, C], C = G groups of Cg channels:
//   z = w (x - mean) rstd + b,   y = act(z)
// with the statistics of every (token, group) (each token for itself: a head norm) or of every
// (sequence, group) of packed sequences.  Backward, with dz = dy act'(z), e = w dz, xh = (x - mean) rstd
// and means over the same elements as the statistics:
//   dx = rstd (e - mean(e) - xh mean(e xh)),   dw = sum dz xh,   db = sum dz
//
// HBM-bound.  Per token: one pass, a group's channels in the registers of a few lanes, statistics by
// shuffles (mean first, then squares about it).  Packed: a pass for the statistics and one for the
// result; the second walks the rows backwards, since the last ~100 MB of the first pass are still in
// L2.  Sums over many rows are kept in 64 bits (squares cancel against the mean) and joined from
// per-chunk parts in a fixed order; nothing is atomic.
#include "common.cuh"
#include "pack_tables.cuh"
#include "vec.cuh"

#include <type_traits>

namespace ssla {
namespace gn {
namespace {

constexpr int TH = 256;
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

enum { ACT_NONE = SSLA_ACT_NONE, ACT_SILU = SSLA_ACT_SILU, ACT_RELU = SSLA_ACT_RELU };

// 1 / (1 + exp(-z)) on the two special-function instructions, each good to about 2^-22: with the
// library's expf and division the instructions, not the memory, bound the kernels (token_fwd of
// 16384 x 4096 bf16: 113 us).  exp(-z) = inf gives 0.
__device__ __forceinline__ float sigmoid(float z) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

template <int ACT> __device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_SILU) return z * sigmoid(z);
  if (ACT == ACT_RELU) return z <= 0.f ? 0.f : z;  // NaN stays
  return z;
}
template <int ACT> __device__ __forceinline__ float act_bwd(float dy, float z) {
  if (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return dy * (s * fmaf(z, 1.f - s, 1.f));
  }
  if (ACT == ACT_RELU) return z <= 0.f ? 0.f : dy;
  return dy;
}
// f(integral constant of the activation): the loops inside carry no test of it
template <class F> __device__ __forceinline__ void with_act(int act, F f) {
  if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
  else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>());
  else f(std::integral_constant<int, ACT_NONE>());
}
// sum over aligned groups of L lanes
__device__ __forceinline__ float lane_sum(float x, int L) {
#pragma unroll
  for (int d = 16; d; d >>= 1)
    if (d < L) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

// VEC elements as they lie in memory: loads for the next token wait in these while this one computes.
template <class TI, int VEC> struct alignas(sizeof(TI) * VEC) Raw {
  TI e[VEC];
};

template <int VEC> __device__ __forceinline__ void load_param(const float* p, int at, float dflt, float* x) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = p ? p[at + i] : dflt;
}

// ------------------------------------------------------------------ one token for itself
// L lanes share a (token, group); every lane keeps NV vectors of VEC channels.  A block's lane
// groups are TP tokens x GB groups; blocks stride over the tokens, so a lane's channels are fixed
// and the backward's dw, db accumulate in registers over its tokens.
struct TokMap {
  int L, GB, TP;  // lanes of a group, groups and tokens of a block
};

template <class TI, int VEC, int NV>
__global__ void __launch_bounds__(TH) token_fwd(const TI* __restrict__ x, int64_t T, int C, int G, TokMap m,
                                                const float* __restrict__ w, const float* __restrict__ b, float eps,
                                                int act, TI* __restrict__ y) {
  griddep_launch_dependents();
  griddep_wait();
  const int Cg = C / G, slot = threadIdx.x / m.L, l = threadIdx.x % m.L;
  const int g = blockIdx.y * m.GB + slot % m.GB, tp = slot / m.GB;
  const bool live = tp < m.TP && g < G;
  const float inv = 1.f / (float)Cg;
  float ww[NV][VEC], bb[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * m.L + l) * VEC;
    if (live && c < Cg) {
      load_param<VEC>(w, g * Cg + c, 1.f, ww[j]);
      load_param<VEC>(b, g * Cg + c, 0.f, bb[j]);
    }
  }
  using R = Raw<TI, VEC>;
  const int64_t step = (int64_t)gridDim.x * m.TP;
  R rx[NV];
  const int64_t first = (int64_t)blockIdx.x * m.TP + tp;
  const TI* px = x + (size_t)first * C + (size_t)g * Cg;
  TI* py = y + (size_t)first * C + (size_t)g * Cg;
  const size_t stride = (size_t)step * C;
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * m.L + l) * VEC;
      if (live && t < T && c < Cg) {
        rx[j] = *reinterpret_cast<const R*>(px + c);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) rx[j].e[i] = TI(0.f);
      }
    }
  };
  fetch(first);
  for (int64_t t0 = (int64_t)blockIdx.x * m.TP; t0 < T; t0 += step, py += stride) {
    const int64_t t = t0 + tp;
    const bool on = live && t < T;
    float v[NV][VEC], s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = ldf(&rx[j].e[i]);
        s += v[j][i];
      }
    px += stride;
    fetch(t + step);
    const float mean = lane_sum(s, m.L) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if ((j * m.L + l) * VEC < Cg)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[j][i] -= mean;
          q = fmaf(v[j][i], v[j][i], q);
        }
    }
    const float rstd = rsqrtf(lane_sum(q, m.L) * inv + eps);
    with_act(act, [&](auto A) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * m.L + l) * VEC;
        if (on && c < Cg) {
          float o[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] = act_fwd<A.value>(fmaf(v[j][i] * rstd, ww[j][i], bb[j][i]));
          Vec<TI, VEC>::store(py + c, o);
        }
      }
    });
  }
}

// part [2][gridDim.x * TP][C]: this block's sums of dz xh and dz over its tokens
constexpr int tok_resident(int per_lane) { return per_lane <= 8 ? 3 : per_lane <= 16 ? 2 : 1; }

template <class TI, int VEC, int NV>
__global__ void __launch_bounds__(TH, tok_resident(VEC * NV)) token_bwd(const TI* __restrict__ x, const TI* __restrict__ dy, int64_t T, int C,
                                                int G, TokMap m, const float* __restrict__ w,
                                                const float* __restrict__ b, float eps, int act, TI* __restrict__ dx,
                                                float* __restrict__ part) {
  griddep_launch_dependents();
  griddep_wait();
  const int Cg = C / G, slot = threadIdx.x / m.L, l = threadIdx.x % m.L;
  const int g = blockIdx.y * m.GB + slot % m.GB, tp = slot / m.GB;
  const bool live = tp < m.TP && g < G;
  const float inv = 1.f / (float)Cg;
  float ww[NV][VEC], bb[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * m.L + l) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = db[j][i] = 0.f;
    if (live && c < Cg) {
      load_param<VEC>(w, g * Cg + c, 1.f, ww[j]);
      load_param<VEC>(b, g * Cg + c, 0.f, bb[j]);
    }
  }
  using R = Raw<TI, VEC>;
  const int64_t step = (int64_t)gridDim.x * m.TP;
  R rx[NV], ry[NV];
  const int64_t first = (int64_t)blockIdx.x * m.TP + tp;
  const size_t start = (size_t)first * C + (size_t)g * Cg, stride = (size_t)step * C;
  const TI *px = x + start, *pd = dy + start;
  TI* po = dx + start;
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * m.L + l) * VEC;
      if (live && t < T && c < Cg) {
        rx[j] = *reinterpret_cast<const R*>(px + c);
        ry[j] = *reinterpret_cast<const R*>(pd + c);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) rx[j].e[i] = ry[j].e[i] = TI(0.f);
      }
    }
  };
  fetch(first);
  for (int64_t t0 = (int64_t)blockIdx.x * m.TP; t0 < T; t0 += step, po += stride) {
    const int64_t t = t0 + tp;
    const bool on = live && t < T;
    float v[NV][VEC], e[NV][VEC], s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = ldf(&rx[j].e[i]);
        e[j][i] = ldf(&ry[j].e[i]);
        s += v[j][i];
      }
    px += stride;
    pd += stride;
    fetch(t + step);
    const float mean = lane_sum(s, m.L) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if ((j * m.L + l) * VEC < Cg)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[j][i] -= mean;
          q = fmaf(v[j][i], v[j][i], q);
        }
    }
    const float rstd = rsqrtf(lane_sum(q, m.L) * inv + eps);
    float s1 = 0.f, s2 = 0.f;
    with_act(act, [&](auto A) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (on && (j * m.L + l) * VEC < Cg)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float xh = v[j][i] * rstd;
            const float dz = act_bwd<A.value>(e[j][i], fmaf(xh, ww[j][i], bb[j][i]));
            dw[j][i] = fmaf(dz, xh, dw[j][i]);
            db[j][i] += dz;
            v[j][i] = xh;
            e[j][i] = dz * ww[j][i];
            s1 += e[j][i];
            s2 = fmaf(e[j][i], xh, s2);
          }
    });
    s1 = lane_sum(s1, m.L) * inv;
    s2 = lane_sum(s2, m.L) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * m.L + l) * VEC;
      if (on && c < Cg) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = rstd * (e[j][i] - s1 - v[j][i] * s2);
        Vec<TI, VEC>::store(po + c, o);
      }
    }
  }
  if (!live) return;
  const size_t rows = (size_t)gridDim.x * m.TP, row = (size_t)blockIdx.x * m.TP + tp;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * m.L + l) * VEC;
    if (c < Cg)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        part[row * C + g * Cg + c + i] = dw[j][i];
        part[(rows + row) * C + g * Cg + c + i] = db[j][i];
      }
  }
}

// out[c] = sum over rows of part[rows][C], blockIdx.y = 0: dw, 1: db
__global__ void __launch_bounds__(1024) column_sums(const float* __restrict__ part, int64_t rows, int C,
                                                    float* __restrict__ dw, float* __restrict__ db) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ double sm[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
  const float* p = part + (blockIdx.y ? (size_t)rows * C : 0);
  double s = 0.0;
  if (c < C)
    for (int64_t r = ty; r < rows; r += 32) s += (double)p[(size_t)r * C + c];
  sm[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < C) {
    s = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sm[i][tx];
    (blockIdx.y ? db : dw)[c] = (float)s;
  }
}

// ------------------------------------------------------------------ packed sequences
// A chunk is up to R tokens of one sequence; a block takes one chunk and a run of whole groups:
// TC column vectors of VEC channels x RP rows at a time.
struct PackMap {
  int R, GB, CV, TC, RP;  // tokens of a chunk; groups and column vectors of a block; threads per row, rows at a time
};

__device__ __forceinline__ bool chunk_at(const longlong2* tab, int64_t c, int64_t& t0, int& rows, int64_t& seq) {
  const longlong2 e = tab[c];
  t0 = e.x;
  rows = (int)(e.y & 0xffffffff);
  seq = e.y >> 32;
  return e.y >= 0;
}

// Four rows at a time, all loads before the first use (one at a time: 40% slower); zeros behind the end.
constexpr int BATCH = 4;
template <class TI, int VEC>
__device__ __forceinline__ void load_batch(Raw<TI, VEC> (&raw)[BATCH], const TI* p, int C, int r, int step, int rows) {
#pragma unroll
  for (int u = 0; u < BATCH; ++u) {
    const int at = r + u * step;
    if (at < rows) raw[u] = *reinterpret_cast<const Raw<TI, VEC>*>(p + (size_t)at * C);
    else
#pragma unroll
      for (int i = 0; i < VEC; ++i) raw[u].e[i] = TI(0.f);
  }
}

// part [MC][G] = (sum x, sum x^2) of the chunk's tokens
template <class TI, int VEC>
__global__ void __launch_bounds__(TH) pack_stats(const TI* __restrict__ x, int C, int G, PackMap m,
                                                 const longlong2* __restrict__ tab, double2* __restrict__ part) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ double2 sm[TH];
  int64_t t0, seq;
  int rows;
  if (!chunk_at(tab, blockIdx.x, t0, rows, seq)) return;
  const int Cg = C / G, g0 = blockIdx.y * m.GB, gn = min(m.GB, G - g0), cv = gn * Cg / VEC;
  const int tc = threadIdx.x % m.TC, rl = threadIdx.x / m.TC;
  double s = 0.0, q = 0.0;
  if (rl < m.RP)
    for (int c = tc; c < cv; c += m.TC) {  // more than one turn only where a block is a single group
      const TI* p = x + (size_t)t0 * C + (size_t)g0 * Cg + c * VEC;
      for (int r = rl; r < rows; r += BATCH * m.RP) {
        Raw<TI, VEC> raw[BATCH];
        load_batch<TI, VEC>(raw, p, C, r, m.RP, rows);
#pragma unroll
        for (int u = 0; u < BATCH; ++u)  // rows behind the end add zeros
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const double d = (double)ldf(&raw[u].e[i]);
            s += d;
            q = fma(d, d, q);
          }
      }
    }
  sm[threadIdx.x] = make_double2(s, q);
  __syncthreads();
  // a group's threads: columns [k CW, (k + 1) CW) of all RP rows
  const int CW = m.GB == 1 ? m.TC : Cg / VEC;
  for (int k = threadIdx.x >> 5; k < gn; k += TH / 32) {  // one warp a group
    double a = 0.0, b = 0.0;
    for (int j = threadIdx.x & 31; j < CW * m.RP; j += 32) {
      const double2 z = sm[(j / CW) * m.TC + k * CW + j % CW];
      a += z.x;
      b += z.y;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, d);
      b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if ((threadIdx.x & 31) == 0) part[(size_t)blockIdx.x * G + g0 + k] = make_double2(a, b);
  }
}

__device__ __forceinline__ int64_t seq_tokens(const int64_t* cu, int64_t n, int64_t T) {
  int64_t b = cu[n], e = cu[n + 1];
  b = b < 0 ? 0 : (b > T ? T : b);
  e = e < b ? b : (e > T ? T : e);
  return e - b;
}

// stats [N][G] = (mean, rstd): one warp per (sequence, group)
__global__ void __launch_bounds__(TH) pack_moments(const double2* __restrict__ part, const int* __restrict__ off,
                                                   const int64_t* __restrict__ cu, int64_t N, int64_t T, int G, int Cg,
                                                   float eps, float2* __restrict__ stats) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t id = (int64_t)blockIdx.x * (TH / 32) + (threadIdx.x >> 5);
  if (id >= N * G) return;
  const int64_t n = id / G;
  const int g = (int)(id - n * G), lane = threadIdx.x & 31;
  double s = 0.0, q = 0.0;
  for (int c = off[n] + lane; c < off[n + 1]; c += 32) {
    const double2 z = part[(size_t)c * G + g];
    s += z.x;
    q += z.y;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, d);
    q += __shfl_xor_sync(0xffffffffu, q, d);
  }
  if (lane) return;
  const double cnt = (double)seq_tokens(cu, n, T) * Cg;
  const double mean = cnt > 0 ? s / cnt : 0.0;
  double var = cnt > 0 ? q / cnt - mean * mean : 0.0;
  var = var < 0.0 ? 0.0 : var;
  stats[id] = make_float2((float)mean, (float)(1.0 / sqrt(var + (double)eps)));
}

template <class TI>
__device__ __forceinline__ void zero_rest(TI* y, const int64_t* cu, int64_t N, int64_t T, int C) {
  int64_t b = cu[0], e = cu[N];
  b = b < 0 ? 0 : (b > T ? T : b);
  e = e < b ? b : (e > T ? T : e);
  const int64_t head = b * C, total = head + (T - e) * C, blocks = (int64_t)gridDim.x * gridDim.y;
  for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * TH + threadIdx.x; i < total; i += blocks * TH)
    y[i < head ? i : e * C + (i - head)] = TI(0.f);
}

template <class TI, int VEC>
__global__ void __launch_bounds__(TH) pack_fwd(const TI* __restrict__ x, int64_t T, int C, int G, PackMap m,
                                               const longlong2* __restrict__ tab, int64_t MC,
                                               const int64_t* __restrict__ cu, int64_t N,
                                               const float2* __restrict__ stats, const float* __restrict__ w,
                                               const float* __restrict__ b, int act, TI* __restrict__ y) {
  griddep_launch_dependents();
  griddep_wait();
  zero_rest(y, cu, N, T, C);
  int64_t t0, seq;
  int rows;
  if (MC == 0 || !chunk_at(tab, MC - 1 - blockIdx.x, t0, rows, seq)) return;  // last rows first: still in L2
  const int Cg = C / G, g0 = blockIdx.y * m.GB, cv = min(m.GB, G - g0) * Cg / VEC;
  const int tc = threadIdx.x % m.TC, rl = threadIdx.x / m.TC;
  if (rl >= m.RP) return;
  for (int c = tc; c < cv; c += m.TC) {
    const int ch = g0 * Cg + c * VEC;
    const float2 st = stats[seq * G + ch / Cg];
    float ww[VEC], bb[VEC];
    load_param<VEC>(w, ch, 1.f, ww);
    load_param<VEC>(b, ch, 0.f, bb);
    const size_t base = (size_t)t0 * C + ch;
    with_act(act, [&](auto A) {
      for (int r = rl; r < rows; r += BATCH * m.RP) {
        Raw<TI, VEC> raw[BATCH];
        load_batch<TI, VEC>(raw, x + base, C, r, m.RP, rows);
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (r + u * m.RP >= rows) break;
          float v[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            v[i] = act_fwd<A.value>(fmaf((ldf(&raw[u].e[i]) - st.x) * st.y, ww[i], bb[i]));
          Vec<TI, VEC>::store(y + base + (size_t)(r + u * m.RP) * C, v);
        }
      }
    });
  }
}

// part [2][MC][C] = a chunk's sums of dz xh and dz
template <class TI, int VEC>
__global__ void __launch_bounds__(TH) pack_sums(const TI* __restrict__ x, const TI* __restrict__ dy, int C, int G,
                                                PackMap m, const longlong2* __restrict__ tab, int64_t MC,
                                                const float2* __restrict__ stats, const float* __restrict__ w,
                                                const float* __restrict__ b, int act, float* __restrict__ part) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ float sm[2][VEC][TH];
  int64_t t0, seq;
  int rows;
  if (!chunk_at(tab, blockIdx.x, t0, rows, seq)) return;
  const int Cg = C / G, g0 = blockIdx.y * m.GB, cv = min(m.GB, G - g0) * Cg / VEC;
  const int tc = threadIdx.x % m.TC, rl = threadIdx.x / m.TC;
  for (int c0 = 0; c0 < cv; c0 += m.TC) {
    const int c = c0 + tc, ch = g0 * Cg + c * VEC;
    const bool in = rl < m.RP && c < cv;
    float dw[VEC], db[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[i] = db[i] = 0.f;
    if (in) {
      const float2 st = stats[seq * G + ch / Cg];
      float ww[VEC], bb[VEC];
      load_param<VEC>(w, ch, 1.f, ww);
      load_param<VEC>(b, ch, 0.f, bb);
      const size_t base = (size_t)t0 * C + ch;
      with_act(act, [&](auto A) {
        for (int r = rl; r < rows; r += BATCH * m.RP) {
          Raw<TI, VEC> rx[BATCH], ry[BATCH];
          load_batch<TI, VEC>(rx, x + base, C, r, m.RP, rows);
          load_batch<TI, VEC>(ry, dy + base, C, r, m.RP, rows);
#pragma unroll
          for (int u = 0; u < BATCH; ++u) {
            if (r + u * m.RP >= rows) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float xh = (ldf(&rx[u].e[i]) - st.x) * st.y;
              const float dz = act_bwd<A.value>(ldf(&ry[u].e[i]), fmaf(xh, ww[i], bb[i]));
              dw[i] = fmaf(dz, xh, dw[i]);
              db[i] += dz;
            }
          }
        }
      });
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sm[0][i][threadIdx.x] = dw[i];
      sm[1][i][threadIdx.x] = db[i];
    }
    __syncthreads();
    if (rl == 0 && c < cv)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float a = 0.f, d = 0.f;
        for (int r = 0; r < m.RP; ++r) {
          a += sm[0][i][r * m.TC + tc];
          d += sm[1][i][r * m.TC + tc];
        }
        part[(size_t)blockIdx.x * C + ch + i] = a;
        part[((size_t)MC + blockIdx.x) * C + ch + i] = d;
      }
  }
}

// seq [2][N][C] = sums of part [2][MC][C] over the chunks of a sequence; 32 channels a block
__global__ void __launch_bounds__(TH) pack_join(const float* __restrict__ part, int64_t MC, const int* __restrict__ off,
                                                int64_t N, int C, float* __restrict__ seq) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ double sm[2][TH / 32][32];
  const int64_t n = blockIdx.x;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.y * 32 + tx;
  double a = 0.0, b = 0.0;
  if (c < C)
    for (int r = off[n] + ty; r < off[n + 1]; r += TH / 32) {
      a += (double)part[(size_t)r * C + c];
      b += (double)part[((size_t)MC + r) * C + c];
    }
  sm[0][ty][tx] = a;
  sm[1][ty][tx] = b;
  __syncthreads();
  if (ty == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < TH / 32; ++i) {
      a += sm[0][i][tx];
      b += sm[1][i][tx];
    }
    seq[(size_t)n * C + c] = (float)a;
    seq[(size_t)(N + n) * C + c] = (float)b;
  }
}

// means [N][G] = (mean e, mean e xh) from the sequences' channel sums: one warp per (sequence, group)
__global__ void __launch_bounds__(TH) pack_means(const float* __restrict__ seq, const int64_t* __restrict__ cu,
                                                 int64_t N, int64_t T, int C, int G, const float* __restrict__ w,
                                                 float2* __restrict__ means) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t id = (int64_t)blockIdx.x * (TH / 32) + (threadIdx.x >> 5);
  if (id >= N * G) return;
  const int64_t n = id / G;
  const int g = (int)(id - n * G), lane = threadIdx.x & 31, Cg = C / G;
  double s1 = 0.0, s2 = 0.0;
  for (int j = lane; j < Cg; j += 32) {
    const int ch = g * Cg + j;
    const double ww = w ? (double)w[ch] : 1.0;
    s2 += ww * (double)seq[(size_t)n * C + ch];
    s1 += ww * (double)seq[(size_t)(N + n) * C + ch];
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s1 += __shfl_xor_sync(0xffffffffu, s1, d);
    s2 += __shfl_xor_sync(0xffffffffu, s2, d);
  }
  if (lane) return;
  const double k = (double)seq_tokens(cu, n, T) * Cg;
  means[id] = k > 0 ? make_float2((float)(s1 / k), (float)(s2 / k)) : make_float2(0.f, 0.f);
}

template <class TI, int VEC>
__global__ void __launch_bounds__(TH) pack_bwd(const TI* __restrict__ x, const TI* __restrict__ dy, int64_t T, int C,
                                               int G, PackMap m, const longlong2* __restrict__ tab, int64_t MC,
                                               const int64_t* __restrict__ cu, int64_t N,
                                               const float2* __restrict__ stats, const float2* __restrict__ means,
                                               const float* __restrict__ w, const float* __restrict__ b, int act,
                                               TI* __restrict__ dx) {
  griddep_launch_dependents();
  griddep_wait();
  zero_rest(dx, cu, N, T, C);
  int64_t t0, seq;
  int rows;
  if (MC == 0 || !chunk_at(tab, MC - 1 - blockIdx.x, t0, rows, seq)) return;
  const int Cg = C / G, g0 = blockIdx.y * m.GB, cv = min(m.GB, G - g0) * Cg / VEC;
  const int tc = threadIdx.x % m.TC, rl = threadIdx.x / m.TC;
  if (rl >= m.RP) return;
  for (int c = tc; c < cv; c += m.TC) {
    const int ch = g0 * Cg + c * VEC;
    const float2 st = stats[seq * G + ch / Cg], mm = means[seq * G + ch / Cg];
    float ww[VEC], bb[VEC];
    load_param<VEC>(w, ch, 1.f, ww);
    load_param<VEC>(b, ch, 0.f, bb);
    const size_t base = (size_t)t0 * C + ch;
    with_act(act, [&](auto A) {
      for (int r = rl; r < rows; r += BATCH * m.RP) {
        Raw<TI, VEC> rx[BATCH], ry[BATCH];
        load_batch<TI, VEC>(rx, x + base, C, r, m.RP, rows);
        load_batch<TI, VEC>(ry, dy + base, C, r, m.RP, rows);
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (r + u * m.RP >= rows) break;
          float v[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float xh = (ldf(&rx[u].e[i]) - st.x) * st.y;
            const float dz = act_bwd<A.value>(ldf(&ry[u].e[i]), fmaf(xh, ww[i], bb[i]));
            v[i] = st.y * (fmaf(dz, ww[i], -mm.x) - xh * mm.y);
          }
          Vec<TI, VEC>::store(dx + base + (size_t)(r + u * m.RP) * C, v);
        }
      }
    });
  }
}

// ------------------------------------------------------------------ host
int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

// Largest vector of a group's channels (16 bytes at most) that its rows allow.
int vec_of(size_t elem, int64_t C, int64_t Cg, const void* const* ptrs, int n) {
  int v = 16 / (int)elem;
  auto ok = [&](int k) {
    if (Cg % k || C % k) return false;
    for (int i = 0; i < n; ++i)
      if (!aligned_to(ptrs[i], k * elem)) return false;
    return true;
  };
  if (ok(v)) return v;
  if (v == 8 && ok(4)) return 4;
  return 1;
}

constexpr int kMaxPerLane = 32;  // channels a lane keeps: groups of up to 1024 channels per token

TokMap tok_map(int64_t Cg, int64_t G, int vec, int* nv) {
  TokMap m;
  const int vecs = (int)(Cg / vec);
  m.L = pow2_at_least(vecs < 32 ? vecs : 32);
  *nv = pow2_at_least((vecs + m.L - 1) / m.L);
  const int lg = TH / m.L;
  m.GB = (int)(G < lg ? G : lg);
  m.TP = lg / m.GB;
  return m;
}

// blocks along the tokens, per_sm on every SM
int tok_blocks(int64_t T, int gy, int TP, int per_sm) {
  int64_t want = (int64_t)kNumSMs * per_sm / gy, most = (T + TP - 1) / TP;
  if (want < 1) want = 1;
  return (int)(want < most ? want : (most > 0 ? most : 1));
}

int chunk_rows(int64_t T, int64_t C) {
  // ~12 blocks per SM even out the last wave; at most 1 MiB of fp32 channels a block
  int64_t r = T / (12 * kNumSMs);
  const int64_t most = 16384 / (C < 16384 ? C : 16384) * 16;
  r = r > most ? most : r;
  r = r < 16 ? 16 : r;
  return (int)r;
}

PackMap pack_map(int64_t T, int64_t C, int64_t G, int vec) {
  PackMap m;
  const int64_t Cg = C / G, gv = Cg / vec;
  m.R = chunk_rows(T, C);
  m.GB = (int)(gv >= TH ? 1 : (TH / gv < G ? TH / gv : G));
  m.CV = (int)(m.GB * gv);
  m.TC = m.CV < TH ? m.CV : TH;
  m.RP = TH / m.TC;
  return m;
}

// What the forward leaves for the backward: the chunk tables and the statistics.
struct PackSaved {
  int* off;
  longlong2* tab;
  float2* stats;
};

size_t pack_saved(void* base, int64_t N, int64_t T, int64_t C, int64_t G, PackSaved* out, int64_t* mc) {
  const int64_t R = chunk_rows(T, C), MC = (T + (R - 1) * N) / R;
  char* q = (char*)base;
  auto take = [&](size_t n) { char* r = q; q += align256(n); return (void*)r; };
  PackSaved s;
  s.off = (int*)take(4 * (N + 1));
  s.tab = (longlong2*)take(16 * (size_t)MC);
  s.stats = (float2*)take(8 * (size_t)N * G);
  if (out) *out = s;
  if (mc) *mc = MC;
  return (size_t)(q - (char*)base);
}

struct PackWork {
  double2* part;   // forward [MC][G]
  float* sums;     // backward [2][MC][C]
  float* seq;      // backward [2][N][C]
  float2* means;   // backward [N][G]
};

size_t pack_work(void* base, int64_t N, int64_t T, int64_t C, int64_t G, bool bwd, PackWork* out) {
  int64_t MC;
  pack_saved(nullptr, N, T, C, G, nullptr, &MC);
  char* q = (char*)base;
  auto take = [&](size_t n) { char* r = q; q += align256(n); return (void*)r; };
  PackWork w;
  w.part = (double2*)take(bwd ? 0 : 16 * (size_t)MC * G);
  w.sums = (float*)take(bwd ? 8 * (size_t)MC * C : 0);
  w.seq = (float*)take(bwd ? 8 * (size_t)N * C : 0);
  w.means = (float2*)take(bwd ? 8 * (size_t)N * G : 0);
  if (out) *out = w;
  return (size_t)(q - (char*)base);
}

size_t tok_part_bytes(int64_t T, int64_t C, int64_t G) {
  // upper bound over the vector widths: blocks * TP rows of C channels, twice
  size_t most = 0;
  for (int vec = 1; vec <= 8; vec *= 2) {
    if ((C / G) % vec) continue;
    int nv;
    const TokMap m = tok_map(C / G, G, vec, &nv);
    const int gy = (int)((G + m.GB - 1) / m.GB);
    const size_t b = (size_t)tok_blocks(T, gy, m.TP, 4) * m.TP * C * 8;
    most = b > most ? b : most;
  }
  return most;
}

int check(const char* name, int dtype, int64_t T, int64_t C, int64_t G, int act, bool packed, int64_t N) {
  SSLA_CHECK_ARG(dtype_ok(dtype), "%s: bad dtype", name);
  SSLA_CHECK_ARG(T >= 0 && N >= 0 && C >= 1 && G >= 1 && C % G == 0, "%s: %lld channels in %lld groups", name,
                 (long long)C, (long long)G);
  SSLA_CHECK_ARG(C <= (1 << 20), "%s: more than 2^20 channels", name);
  SSLA_CHECK_ARG(act >= ACT_NONE && act <= ACT_RELU, "%s: bad activation", name);
  SSLA_CHECK_ARG(packed || C / G <= 32 * kMaxPerLane, "%s: per token, a group has at most %d channels", name,
                 32 * kMaxPerLane);
  SSLA_CHECK_ARG(T < (int64_t(1) << 31) && N < (int64_t(1) << 31) && N * G < (int64_t(1) << 33), "%s: too many rows", name);
  return SSLA_OK;
}

struct Call {
  const void *x, *dy;
  int64_t T, N;
  int C, G;
  const float *w, *b;
  float eps;
  int act;
  const int64_t* cu;
  void* y;  // or dx
  void* saved;
  float *dw, *db;
  void* ws;
};

template <class TI, int VEC, int NV> int token_call(const Call& c, const TokMap& m, cudaStream_t st) {
  const int gy = (c.G + m.GB - 1) / m.GB;
  if (!c.dy) {
    launch_pdl(token_fwd<TI, VEC, NV>, dim3(tok_blocks(c.T, gy, m.TP, 32), gy), dim3(TH), 0, st, (const TI*)c.x, c.T, c.C, c.G, m, c.w, c.b, c.eps, c.act, (TI*)c.y);
    SSLA_CHECK_LAUNCH("group_norm forward");
    return SSLA_OK;
  }
  const int gx = tok_blocks(c.T, gy, m.TP, tok_resident(VEC * NV));  // one wave: the sums stay in registers
  launch_pdl(token_bwd<TI, VEC, NV>, dim3(gx, gy), dim3(TH), 0, st, (const TI*)c.x, (const TI*)c.dy, c.T, c.C, c.G, m, c.w, c.b, c.eps,
                                                      c.act, (TI*)c.y, (float*)c.ws);
  SSLA_CHECK_LAUNCH("group_norm backward");
  launch_pdl(column_sums, dim3((c.C + 31) / 32, 2), dim3(1024), 0, st, (const float*)c.ws, (int64_t)gx * m.TP, c.C, c.dw, c.db);
  SSLA_CHECK_LAUNCH("group_norm column sums");
  return SSLA_OK;
}

template <class TI, int VEC> int token_vec(const Call& c, cudaStream_t st) {
  int nv;
  const TokMap m = tok_map(c.C / c.G, c.G, VEC, &nv);
#define SSLA_GN_NV(n) \
  if constexpr (n * VEC <= kMaxPerLane) { if (nv == n) return token_call<TI, VEC, n>(c, m, st); }
  SSLA_GN_NV(1)
  SSLA_GN_NV(2)
  SSLA_GN_NV(4)
  SSLA_GN_NV(8)
  SSLA_GN_NV(16)
  SSLA_GN_NV(32)
#undef SSLA_GN_NV
  set_error("group_norm: groups of %d channels are too wide", c.C / c.G);
  return SSLA_ERR_UNSUPPORTED;
}

template <class TI, int VEC> int pack_call(const Call& c, cudaStream_t st) {
  PackSaved sv;
  PackWork w;
  int64_t MC;
  pack_saved(c.saved, c.N, c.T, c.C, c.G, &sv, &MC);
  pack_work(c.ws, c.N, c.T, c.C, c.G, c.dy != nullptr, &w);
  const PackMap m = pack_map(c.T, c.C, c.G, VEC);
  const dim3 grid((unsigned)(MC > 0 ? MC : 1), (c.G + m.GB - 1) / m.GB);
  const unsigned ngrid = (unsigned)((c.N * c.G + TH / 32 - 1) / (TH / 32));
  if (!c.dy) {
    int rc = launch_pack_tables(c.cu, c.N, c.T, m.R, MC, sv.off, sv.tab, st);
    if (rc) return rc;
    if (MC > 0) {
      launch_pdl(pack_stats<TI, VEC>, grid, dim3(TH), 0, st, (const TI*)c.x, c.C, c.G, m, sv.tab, w.part);
      SSLA_CHECK_LAUNCH("group_norm statistics");
    }
    if (ngrid) {
      launch_pdl(pack_moments, dim3(ngrid), dim3(TH), 0, st, w.part, sv.off, c.cu, c.N, c.T, c.G, c.C / c.G, c.eps, sv.stats);
      SSLA_CHECK_LAUNCH("group_norm moments");
    }
    if (c.T == 0) return SSLA_OK;
    launch_pdl(pack_fwd<TI, VEC>, grid, dim3(TH), 0, st, (const TI*)c.x, c.T, c.C, c.G, m, sv.tab, MC, c.cu, c.N, sv.stats, c.w, c.b,
                                           c.act, (TI*)c.y);
    SSLA_CHECK_LAUNCH("group_norm forward");
    return SSLA_OK;
  }
  if (MC > 0) {
    launch_pdl(pack_sums<TI, VEC>, grid, dim3(TH), 0, st, (const TI*)c.x, (const TI*)c.dy, c.C, c.G, m, sv.tab, MC, sv.stats, c.w, c.b,
                                            c.act, w.sums);
    SSLA_CHECK_LAUNCH("group_norm sums");
  }
  if (c.N > 0) {
    launch_pdl(pack_join, dim3((unsigned)c.N, (c.C + 31) / 32), dim3(TH), 0, st, w.sums, MC, sv.off, c.N, c.C, w.seq);
    SSLA_CHECK_LAUNCH("group_norm join");
  }
  launch_pdl(column_sums, dim3((c.C + 31) / 32, 2), dim3(1024), 0, st, w.seq, c.N, c.C, c.dw, c.db);
  SSLA_CHECK_LAUNCH("group_norm column sums");
  if (ngrid) {
    launch_pdl(pack_means, dim3(ngrid), dim3(TH), 0, st, w.seq, c.cu, c.N, c.T, c.C, c.G, c.w, w.means);
    SSLA_CHECK_LAUNCH("group_norm means");
  }
  if (c.T == 0) return SSLA_OK;
  launch_pdl(pack_bwd<TI, VEC>, grid, dim3(TH), 0, st, (const TI*)c.x, (const TI*)c.dy, c.T, c.C, c.G, m, sv.tab, MC, c.cu, c.N,
                                         sv.stats, w.means, c.w, c.b, c.act, (TI*)c.y);
  SSLA_CHECK_LAUNCH("group_norm backward");
  return SSLA_OK;
}

int dispatch(const Call& c, int dtype, cudaStream_t st) {
  return SSLA_DISPATCH_DTYPE(dtype, T_, [&] {
    const void* ptrs[3] = {c.x, c.y, c.dy};
    const int vec = vec_of(sizeof(T_), c.C, c.C / c.G, ptrs, 3);
    if constexpr (sizeof(T_) == 2) {
      if (vec == 8) return c.cu ? pack_call<T_, 8>(c, st) : token_vec<T_, 8>(c, st);
    }
    if (vec == 4) return c.cu ? pack_call<T_, 4>(c, st) : token_vec<T_, 4>(c, st);
    return c.cu ? pack_call<T_, 1>(c, st) : token_vec<T_, 1>(c, st);
  });
}

}  // namespace
}  // namespace gn
}  // namespace ssla

using namespace ssla;
using namespace ssla::gn;

extern "C" size_t ssla_group_norm_act_saved_bytes(int64_t T, int64_t C, int64_t G, int64_t n_seqs) {
  if (T < 0 || C < 1 || G < 1 || C % G || n_seqs < 0) return 0;
  return pack_saved(nullptr, n_seqs, T, C, G, nullptr, nullptr);
}

extern "C" size_t ssla_group_norm_act_workspace_bytes(int64_t T, int64_t C, int64_t G, int packed, int64_t n_seqs,
                                                      int backward) {
  if (T < 0 || C < 1 || G < 1 || C % G || n_seqs < 0) return 0;
  if (packed) return pack_work(nullptr, n_seqs, T, C, G, backward != 0, nullptr);
  return backward ? tok_part_bytes(T, C, G) : 0;
}

// Buffers of one call: the workspace, and with cu_seqlens what the forward saves.
static int check_buffers(const char* name, int64_t T, int64_t C, int64_t G, bool packed, int64_t N, bool bwd,
                         const void* saved, size_t saved_bytes, const void* ws, size_t ws_bytes) {
  const size_t need = ssla_group_norm_act_workspace_bytes(T, C, G, packed, N, bwd);
  const size_t keep = packed ? ssla_group_norm_act_saved_bytes(T, C, G, N) : 0;
  if (ws_bytes < need || (need && !ws) || saved_bytes < keep || (keep && !saved)) {
    set_error("%s: saved buffer of %zu bytes and workspace of %zu, %zu and %zu needed", name, saved_bytes, ws_bytes, keep,
              need);
    return SSLA_ERR_WORKSPACE;
  }
  SSLA_CHECK_ARG(aligned_to(ws, 16) && aligned_to(saved, 16), "%s: misaligned workspace or saved buffer", name);
  return SSLA_OK;
}

extern "C" int ssla_group_norm_act_fwd(const void* x, int dtype, int64_t T, int64_t C, int64_t G, const float* w,
                                       const float* b, float eps, int act, const int64_t* cu_seqlens, int64_t n_seqs,
                                       void* y, void* saved, size_t saved_bytes, void* workspace,
                                       size_t workspace_bytes, ssla_stream_t stream) {
  const char* name = "ssla_group_norm_act_fwd";
  int rc = check(name, dtype, T, C, G, act, cu_seqlens != nullptr, n_seqs);
  if (rc) return rc;
  if (T == 0 && (!cu_seqlens || n_seqs == 0)) return SSLA_OK;
  SSLA_CHECK_ARG(T == 0 || (x && y), "%s: null pointer", name);
  if ((rc = check_buffers(name, T, C, G, cu_seqlens != nullptr, n_seqs, false, saved, saved_bytes, workspace,
                          workspace_bytes)))
    return rc;
  const Call c = {x, nullptr, T, n_seqs, (int)C, (int)G, w, b, eps, act, cu_seqlens, y, saved, nullptr, nullptr, workspace};
  return dispatch(c, dtype, (cudaStream_t)stream);
}

extern "C" int ssla_group_norm_act_bwd(const void* x, const void* dy, int dtype, int64_t T, int64_t C, int64_t G,
                                       const float* w, const float* b, float eps, int act, const int64_t* cu_seqlens,
                                       int64_t n_seqs, const void* saved, size_t saved_bytes, void* dx, float* dw,
                                       float* db, void* workspace, size_t workspace_bytes, ssla_stream_t stream) {
  const char* name = "ssla_group_norm_act_bwd";
  int rc = check(name, dtype, T, C, G, act, cu_seqlens != nullptr, n_seqs);
  if (rc) return rc;
  SSLA_CHECK_ARG(dw && db && (T == 0 || (x && dy && dx)), "%s: null pointer", name);
  if ((rc = check_buffers(name, T, C, G, cu_seqlens != nullptr, n_seqs, true, saved, saved_bytes, workspace,
                          workspace_bytes)))
    return rc;
  // dy marks the backward for the dispatch, also where there are no rows
  const Call c = {x, dy ? dy : dw, T, n_seqs, (int)C, (int)G, w, b, eps, act, cu_seqlens, dx, const_cast<void*>(saved),
                  dw, db, workspace};
  return dispatch(c, dtype, (cudaStream_t)stream);
}
