// Gated delta rule token by token (fused_recurrent_gated_delta_rule forward), the serving path:
//   S <- exp(g) S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q
//
// A single token is bound by HBM: the fp32 state [K, V] is read and written once, the token's
// vectors are small.  One warp owns a 32-column slice of one (sequence, value head) state: lane
// 8 r + c keeps rows r, r + 4, ... of columns [4c, 4c+4) as float4 registers, so every load of a
// warp takes four neighbouring 128-byte row pieces (rows a quarter of K apart: 5% slower at K = 32)
// and all of a slice's loads are in flight at once.
// Both products with the state are formed in one pass over the registers before the update,
//   S_new^T q = exp(g) S^T q + (k.q) u,
// which leaves one reduction over the four row groups per token (two shuffles) in the token's
// dependent chain.  k and q wait in shared memory, private to the warp.
#include "delta_rule.cuh"

namespace ssla {
namespace delta {
namespace {

constexpr int RWARPS = 2;  // small blocks leave their place to the next one early: 4 warps 2-5% slower

template <class TI, int KP, int RG, bool VEC>
__device__ __forceinline__ void recurrent_warp(const Args& a, const float* __restrict__ h0, TI* __restrict__ o,
                                               float* __restrict__ ht, float* tok) {
  constexpr int KR = KP / RG, LD = KR + 4;  // the pad keeps the row groups on different banks
  constexpr bool STREAM = KP > 64;  // evict-first: 198 us against 225 for 8192 states of 128 x 128, but 418
                                    // against 394 for 262144 of 32 x 32
  constexpr int CL = 32 / RG, COLS = 4 * CL;  // lanes of a row, columns of a warp
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const unsigned slices = (unsigned)(a.V + COLS - 1) / COLS;
  const unsigned warp = blockIdx.x * RWARPS + wid;
  const unsigned sh = warp / slices;
  if (sh >= (unsigned)(a.N * a.HV)) return;
  const unsigned seq = sh / (unsigned)a.HV;
  const int hv = (int)(sh - seq * a.HV), h = hv / a.R;
  const int r = lane / CL, col = (int)(warp - sh * slices) * COLS + (lane % CL) * 4;
  int64_t t0 = a.cu[seq], t1 = a.cu[seq + 1];
  t0 = t0 < 0 ? 0 : (t0 > a.T ? a.T : t0);
  t1 = t1 < t0 ? t0 : (t1 > a.T ? a.T : t1);

  float S[KR][4];
  const size_t base = (size_t)sh * a.K * a.V + col;
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int row = RG * i + r;
    S[i][0] = S[i][1] = S[i][2] = S[i][3] = 0.f;
    if (h0 && row < a.K) {
      const float* p = h0 + base + (size_t)row * a.V;
      if (VEC) {
        if (col < a.V) {
          const float4* q4 = reinterpret_cast<const float4*>(p);
          const float4 x = STREAM ? __ldcs(q4) : __ldg(q4);
          S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (col + c < a.V) S[i][c] = p[c];
      }
    }
  }
  float* sk = tok;
  float* sq = tok + RG * LD;
  for (int64_t t = t0; t < t1; ++t) {
    const size_t kb = ((size_t)t * a.H + h) * a.K, vb = ((size_t)t * a.HV + hv) * a.V + col;
    float kq = 0.f;
    __syncwarp();
#pragma unroll
    for (int i = lane; i < KP; i += 32) {
      float x = 0.f, y = 0.f;
      if (i < a.K) {
        x = ldf((const TI*)a.k + kb + i);
        y = ldf((const TI*)a.q + kb + i);
      }
      const int at = (i % RG) * LD + i / RG;
      sk[at] = x;
      sq[at] = y;
      kq = fmaf(x, y, kq);
    }
    const float d = expf(ld_any(a.g, a.dt_g, (size_t)t * a.HV + hv));
    const float beta = ld_any(a.beta, a.dt_b, (size_t)t * a.HV + hv);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (col + c < a.V) v[c] = ldf((const TI*)a.v + vb + c);
    __syncwarp();
    float pk[4] = {0.f, 0.f, 0.f, 0.f}, pq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KR; i += 4) {
      const float4 k4 = *reinterpret_cast<const float4*>(sk + r * LD + i);
      const float4 q4 = *reinterpret_cast<const float4*>(sq + r * LD + i);
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          pk[c] = fmaf(kk[j], S[i + j][c], pk[c]);
          pq[c] = fmaf(qq[j], S[i + j][c], pq[c]);
        }
    }
#pragma unroll
    for (int m = CL; m <= 16; m <<= 1)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        pk[c] += __shfl_xor_sync(0xffffffffu, pk[c], m);
        pq[c] += __shfl_xor_sync(0xffffffffu, pq[c], m);
      }
#pragma unroll
    for (int m = 16; m; m >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, m);
    float u[4], out[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u[c] = beta * (v[c] - d * pk[c]);
      out[c] = a.scale * fmaf(kq, u[c], d * pq[c]);
    }
#pragma unroll
    for (int i = 0; i < KR; i += 4) {
      const float4 k4 = *reinterpret_cast<const float4*>(sk + r * LD + i);
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) S[i + j][c] = fmaf(kk[j], u[c], d * S[i + j][c]);
    }
    if (r == 0) {
      if (VEC) {
        if (col < a.V) Vec<TI, 4>::store(o + vb, out);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (col + c < a.V) stf(o + vb + c, out[c]);
      }
    }
  }
  if (!ht) return;
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int row = RG * i + r;
    if (row >= a.K) continue;
    float* p = ht + base + (size_t)row * a.V;
    if (VEC) {
      const float4 x = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
      if (col < a.V) {
        if (STREAM) __stcs(reinterpret_cast<float4*>(p), x);
        else *reinterpret_cast<float4*>(p) = x;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < a.V) p[c] = S[i][c];
    }
  }
}

// Resident blocks: as many as the state's registers leave (14 blocks at K = 32 keep 112 KB of loads in
// flight; fewer registers spill, fewer blocks lose 4-15%).
template <class TI, int KP, int RG, bool VEC>
__global__ void __launch_bounds__(RWARPS * 32, KP <= 32 ? 14 : KP == 64 ? 8 : 4) recurrent_kernel(Args a, const float* __restrict__ h0, TI* __restrict__ o,
                                                                float* __restrict__ ht) {
  __shared__ __align__(16) float tok[RWARPS][2 * RG * (KP / RG + 4)];
  recurrent_warp<TI, KP, RG, VEC>(a, h0, o, ht, tok[threadIdx.x >> 5]);
  zero_uncovered(o, a, (int64_t)a.HV * a.V);
}

template <class TI, int KP, int RG>
int launch(const Args& a, const float* h0, void* o, float* ht, cudaStream_t st) {
  constexpr int COLS = 128 / RG;
  const int64_t warps = a.N * a.HV * ((a.V + COLS - 1) / COLS);
  const unsigned grid = (unsigned)((warps + RWARPS - 1) / RWARPS);
  const bool vec = a.V % 4 == 0 && aligned_to(h0, 16) && aligned_to(ht, 16) && aligned_to(o, 4 * sizeof(TI));
  if (vec) recurrent_kernel<TI, KP, RG, true><<<grid ? grid : 1, RWARPS * 32, 0, st>>>(a, h0, (TI*)o, ht);
  else recurrent_kernel<TI, KP, RG, false><<<grid ? grid : 1, RWARPS * 32, 0, st>>>(a, h0, (TI*)o, ht);
  SSLA_CHECK_LAUNCH("ssla_recurrent_gated_delta_rule_fwd");
  return SSLA_OK;
}

}  // namespace
}  // namespace delta
}  // namespace ssla

using namespace ssla;
using namespace ssla::delta;

extern "C" int ssla_recurrent_gated_delta_rule_fwd(const void* q, const void* k, const void* v, const void* g,
                                                   const void* beta, int dtype, int dtype_g, int dtype_beta,
                                                   const int64_t* cu_seqlens, int64_t n_seqs, int64_t T, int64_t H,
                                                   int64_t HV, int64_t K, int64_t V, float scale, const float* h0,
                                                   void* o, float* ht, ssla_stream_t stream) {
  const char* name = "ssla_recurrent_gated_delta_rule_fwd";
  SSLA_CHECK_ARG(dtype_ok(dtype) && dtype_ok(dtype_g) && dtype_ok(dtype_beta), "%s: bad dtype", name);
  SSLA_CHECK_ARG(n_seqs >= 0 && T >= 0 && H >= 0 && HV >= 0, "%s: negative size", name);
  SSLA_CHECK_ARG(H > 0 ? HV % H == 0 : HV == 0, "%s: %lld value heads over %lld key heads", name, (long long)HV,
                 (long long)H);
  SSLA_CHECK_ARG(K >= 1 && V >= 1 && K <= 128 && V <= 256, "%s: K=%lld V=%lld not supported (1 <= K <= 128, 1 <= V <= 256)",
                 name, (long long)K, (long long)V);
  SSLA_CHECK_ARG(n_seqs < (int64_t(1) << 28) && n_seqs * HV < (int64_t(1) << 28), "%s: too many states (%lld x %lld)",
                 name, (long long)n_seqs, (long long)HV);
  if (HV == 0) return SSLA_OK;
  SSLA_CHECK_ARG(cu_seqlens, "%s: null cu_seqlens", name);
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && o), "%s: null pointer", name);
  if (n_seqs == 0 && T == 0) return SSLA_OK;
  cudaStream_t st = (cudaStream_t)stream;
  const Args a = make_args(q, k, v, g, beta, dtype, dtype_g, dtype_beta, cu_seqlens, n_seqs, T, H, HV, K, V, scale);
  return SSLA_DISPATCH_DTYPE(dtype, T_, [&] {
    if (K <= 16) return launch<T_, 16, 4>(a, h0, o, ht, st);
    if (K <= 32) return launch<T_, 32, 4>(a, h0, o, ht, st);
    if (K <= 64) return launch<T_, 64, 4>(a, h0, o, ht, st);
    return launch<T_, 128, 4>(a, h0, o, ht, st);
  });
}
