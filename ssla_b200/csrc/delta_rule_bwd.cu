// Chunked gated delta rule, backward (the kernels here: fp32 tokens; 16-bit ones: delta_rule_16_bwd.cu).
// With P = G o Q K^T (lower), S the state at a chunk's start,
// D the adjoint of the state at its end, X = V - exp(gc) K S, U = T beta X:
//   adjoint of the chunk map   dB = scale qh^T dO,  qh = exp(gc) Q - P W,  W = T beta exp(gc) K
//   dU = scale P^T dO + Kl D;  F = T^T dU;  dV = beta F
//   dP = scale (dO U^T) o G (lower),  E = (F U^T) o G (strictly lower)
//   dQ = scale exp(gc) dO S^T + dP K
//   dK = [-beta exp(gc) F S^T - beta E K] + [exp(gC - gc) U D^T + dP^T Q - E^T beta K]
//   dbeta_i = F_i . X_i - k_i . (E K)_i
// The first bracket of dK is K's part as the row (later) index of the scores, the second as the
// column; every decay exp(gc_i - gc_j) pairs a row i with a column j and adds the pair's term to dg of
// the tokens between, j < t <= i (the chunk's start is the column of the terms with S, its end the row of
// those with D).  So with r_i = q_i . dq_i + k_i . dk_i[row], c_i = k_i . dk_i[column] without the
// terms with D, and l_i = k_i . (exp(gC - gc) U D^T)_i,
//   dg_t = sum_{i >= t} (r_i - c_i) + sum_{i < t} l_i + exp(gC) <S, D>.
// The pairs behind t cancel in the first sum.  The diagonal of dP, a decay of 1 between a token and
// itself, belongs to no dg, but is by far the largest term where a head forgets fast: it stays out of dP
// (strictly lower here) and joins dq and dk behind the sums, q_i k_i dP_ii each.  With it inside, dg at
// g = -20 was its rounding alone.
#include "delta_rule.cuh"

namespace ssla {
namespace delta {
namespace {

using TI = float;  // 16-bit tokens: delta_rule_16_bwd.cu

template <int KP> struct AdjSmem {
  static constexpr int LDK = KP + 8, LDW = KP + 4, LDO = 72;
  TI k[BT * LDK];
  TI q[BT * LDK];
  TI d[BT * LDO];
  float p[BT * LDC];
  float t[BT * LDC];
  float w[BT * LDW];
  Gates gates;
};

// dB of every (chunk, value head).
template <int KP>
__global__ void __launch_bounds__(THREADS, sizeof(AdjSmem<KP>) <= 113 * 1024 ? 2 : 1)
    adjoint_kernel(Args a, const longlong2* __restrict__ tab, int VP, const float* __restrict__ tinv,
                   const TI* __restrict__ dout, float* __restrict__ inc) {
  griddep_launch_dependents();
  griddep_wait();
  using S = AdjSmem<KP>;
  constexpr int LDK = S::LDK, LDW = S::LDW, LDO = S::LDO, NK = KP / 16;
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
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V;
  const bool vec_d = a.vec_v && (reinterpret_cast<uintptr_t>(dout) & 15) == 0;
  load_rows<TI, LDO, 64>(s.d, dout + vo, (size_t)a.HV * a.V, rows, a.V, vec_d);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  cp_wait<0>();
  __syncthreads();
  const TI *sk = s.k, *sq = s.q;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32, k0 = (warp & 1) * (KP / 2);
  {
    float acc[1][4][4];
    zero(acc);
    if (n0 <= m0)
      warp_mma(acc, m0, n0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); },
                         [&](int k, int n) { return pair(sk + n * LDK + k); });
    fade_scores<false, false>(acc, s.gates, m0, n0);
    each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
      *reinterpret_cast<float2*>(s.p + i * LDC + j) = make_float2(x, y);
    });
  }
  float acc[1][NK][4];
  zero(acc);
  warp_mma(acc, m0, k0, 0, m0 + 16,
                         [&](int i, int j) {
                           const float2 x = pair(s.t + i * LDC + j), b = pair(s.gates.beta + j), e = pair(s.gates.start + j);
                           return make_float2(x.x * (b.x * e.x), x.y * (b.y * e.y));
                         },
                         [&](int j, int n) { return column<LDK>(sk + j * LDK + n); });
  each_pair(acc, m0, k0, [&](int i, int n, float x, float y) {
    *reinterpret_cast<float2*>(s.w + i * LDW + n) = make_float2(x, y);
  });
  __syncthreads();
  zero(acc);
  warp_mma(acc, m0, k0, 0, m0 + 16, [&](int i, int j) { return pair(s.p + i * LDC + j); },
                         [&](int j, int n) { return column<LDW>(s.w + j * LDW + n); });
  __syncthreads();
  each_pair(acc, m0, k0, [&](int i, int n, float x, float y) {
    const float e = s.gates.start[i];
    *reinterpret_cast<float2*>(s.w + i * LDW + n) =
        make_float2(a.scale * (e * ldf(sq + i * LDK + n) - x), a.scale * (e * ldf(sq + i * LDK + n + 1) - y));
  });
  constexpr int MT = KP / 64;
  const int mk = (warp >> 1) * 16 * MT;
  for (int v0 = 0; v0 < VP; v0 += 64) {
    if (v0) {
      __syncthreads();
      load_rows<TI, LDO, 64>(s.d, dout + vo + v0, (size_t)a.HV * a.V, rows, a.V - v0, vec_d);
      cp_commit();
      cp_wait<0>();
    }
    __syncthreads();
    float db[MT][4][4];
    zero(db);
    warp_mma(db, mk, n0, 0, BT, [&](int m, int j) { return column<LDW>(s.w + j * LDW + m); },
                         [&](int j, int n) { return column<LDO>(s.d + j * LDO + n); });
    each_pair(db, mk, n0, [&](int m, int n, float x, float y) {
      *reinterpret_cast<float2*>(inc_at(inc, item, KP, VP, m, v0 + n)) = make_float2(x, y);
    });
  }
}

template <int KP> struct BwdSmem {
  // p and t, s and e are read both along rows and down columns: one of the two conflicts either way
  static constexpr int VB = 32, LDK = KP + 8, LDO = VB + 8, LDX = VB + 8, LDS = VB + 4, LDP = BT + 4;
  TI k[BT * LDK];
  TI q[BT * LDK];
  TI d[BT * LDO];
  float p[BT * LDP];  // P, then dP
  float t[BT * LDP];  // T, then E
  float x[BT * LDX];  // beta X, then U
  float f[BT * LDX];  // dU, then F
  float s[KP * LDS];
  float e[KP * LDS];  // D
  float red[6][2][BT];
  float dots[THREADS / 32];
  float diag[BT];  // of dP
  Gates gates;
};

template <int KP>
__device__ __forceinline__ void backward_chunk(const Args& a, const longlong2* __restrict__ tab, int VP,
                                               const float* __restrict__ tinv, const float* __restrict__ states,
                                               const float* __restrict__ ds, const TI* __restrict__ dout,
                                               TI* __restrict__ dq, TI* __restrict__ dk, TI* __restrict__ dv,
                                               void* __restrict__ dg, void* __restrict__ dbeta,
                                               float* __restrict__ dqk) {
  using S = BwdSmem<KP>;
  constexpr int VB = S::VB, LDK = S::LDK, LDO = S::LDO, LDX = S::LDX, LDS = S::LDS, LDP = S::LDP, NT = VB / 16, NK = KP / 16;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const size_t TK = (size_t)a.T * a.HV * a.K;
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const size_t qk = ((size_t)t0 * a.H + h) * a.K;
  load_rows<TI, LDK, KP>(s.k, (const TI*)a.k + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_rows<TI, LDK, KP>(s.q, (const TI*)a.q + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_f32<LDP, BT, BT>(s.t, tinv + item * (BT * BT), BT);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  const TI *sk = s.k, *sq = s.q, *sd = s.d;
  const int m0 = (warp >> 1) * 16, half = warp & 1, n0 = half * (VB / 2), p0 = half * 32, k0 = half * (KP / 2);
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V, vstride = (size_t)a.HV * a.V;
  const bool vec_d = a.vec_v && (reinterpret_cast<uintptr_t>(dout) & 15) == 0;
  const TI* gv = (const TI*)a.v + vo;
  auto fk_row = [&](int m, int k) { return pair(sk + m * LDK + k); };
  auto fx = [&](int k, int n) { return column<LDX>(s.x + k * LDX + n); };

  float aq[1][NK][4], ar[1][NK][4], ac[1][NK][4];  // dO S^T, F S^T, U D^T
  float ap[1][4][4], ae[1][4][4];                  // dO U^T, F U^T
  zero(aq); zero(ar); zero(ac); zero(ap); zero(ae);
  float rb[2] = {0.f, 0.f};  // F . X of rows m0 + lane/4 (+ 8)
  float dot = 0.f;           // <S, D>
  const bool low = p0 <= m0;
  for (int v0 = 0; v0 < a.V; v0 += VB) {
    __syncthreads();
    load_f32<LDS, KP, VB>(s.s, states + item * KP * VP + v0, VP);
    load_f32<LDS, KP, VB>(s.e, ds + item * KP * VP + v0, VP);
    load_rows<TI, LDO, VB>(s.d, dout + vo + v0, vstride, rows, a.V - v0, vec_d);
    cp_commit();
    if (v0 == 0) {
      cp_wait<1>();
      __syncthreads();
      float acc[1][4][4];
      zero(acc);
      if (low)
        warp_mma(acc, m0, p0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); },
                           [&](int k, int n) { return pair(sk + n * LDK + k); });
      fade_scores<false, false>(acc, s.gates, m0, p0);
      each_pair(acc, m0, p0, [&](int i, int j, float x, float y) {
        *reinterpret_cast<float2*>(s.p + i * LDP + j) = make_float2(x, y);
      });
    }
    float xv[1][NT][4];
    each_pair(xv, m0, n0, [&](int i, int n, float& x, float& y) {
      const int c = v0 + n;
      x = i < rows && c < a.V ? ldf(gv + i * vstride + c) : 0.f;
      y = i < rows && c + 1 < a.V ? ldf(gv + i * vstride + c + 1) : 0.f;
    });
    cp_wait<0>();
    __syncthreads();
    float ks[1][NT][4], du[1][NT][4];
    zero(ks);
    zero(du);
    warp_mma(ks, m0, n0, 0, KP, fk_row, [&](int k, int n) { return column<LDS>(s.s + k * LDS + n); });
    warp_mma(du, m0, n0, 0, KP, fk_row, [&](int k, int n) { return column<LDS>(s.e + k * LDS + n); });
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = m0 + (lane >> 2) + (r >= 2 ? 8 : 0);
        xv[0][j][r] -= s.gates.start[i] * ks[0][j][r];
        du[0][j][r] *= s.gates.left[i];
      }
    each_pair(xv, m0, n0, [&](int i, int n, float x, float y) {
      const float b = s.gates.beta[i];
      *reinterpret_cast<float2*>(s.x + i * LDX + n) = make_float2(b * x, b * y);
    });
    for (int i = tid; i < KP * (VB / 4); i += THREADS) {
      const int r = i / (VB / 4), c = (i % (VB / 4)) * 4;
      const float4 x = *reinterpret_cast<const float4*>(s.s + r * LDS + c);
      const float4 y = *reinterpret_cast<const float4*>(s.e + r * LDS + c);
      dot += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
    }
    __syncthreads();
    zero(ks);
    warp_mma(ks, m0, n0, 0, m0 + 16, [&](int m, int k) { return pair(s.t + m * LDP + k); }, fx);  // U
    {
      float pd[1][NT][4];
      zero(pd);
      warp_mma(pd, m0, n0, m0, BT, [&](int m, int k) { return column<LDP>(s.p + k * LDP + m); },
                           [&](int k, int n) { return column<LDO>(sd + k * LDO + n); });
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) du[0][j][r] = fmaf(a.scale, pd[0][j][r], du[0][j][r]);
    }
    __syncthreads();
    each_pair(ks, m0, n0, [&](int i, int n, float x, float y) {
      *reinterpret_cast<float2*>(s.x + i * LDX + n) = make_float2(x, y);
    });
    each_pair(du, m0, n0, [&](int i, int n, float x, float y) {
      *reinterpret_cast<float2*>(s.f + i * LDX + n) = make_float2(x, y);
    });
    __syncthreads();
    zero(du);
    warp_mma(du, m0, n0, m0, BT, [&](int m, int k) { return column<LDP>(s.t + k * LDP + m); },
                             [&](int k, int n) { return column<LDX>(s.f + k * LDX + n); });  // F
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      rb[0] += du[0][j][0] * xv[0][j][0] + du[0][j][1] * xv[0][j][1];
      rb[1] += du[0][j][2] * xv[0][j][2] + du[0][j][3] * xv[0][j][3];
    }
    each_pair(du, m0, n0, [&](int i, int n, float x, float y) {
      const int c = v0 + n;
      if (i < rows) {
        const float b = s.gates.beta[i];
        TI* p = dv + vo + i * vstride + c;
        if (c < a.V) stf(p, b * x);
        if (c + 1 < a.V) stf(p + 1, b * y);
      }
    });
    __syncthreads();
    each_pair(du, m0, n0, [&](int i, int n, float x, float y) {
      *reinterpret_cast<float2*>(s.f + i * LDX + n) = make_float2(x, y);
    });
    __syncthreads();
    auto ff = [&](int m, int k) { return pair(s.f + m * LDX + k); };
    auto fd = [&](int m, int k) { return pair(sd + m * LDO + k); };
    auto fu_t = [&](int k, int n) { return pair(s.x + n * LDX + k); };
    auto fs_t = [&](int k, int n) { return pair(s.s + n * LDS + k); };
    if (low) {
      warp_mma(ap, m0, p0, 0, VB, fd, fu_t);
      warp_mma(ae, m0, p0, 0, VB, ff, fu_t);
    }
    warp_mma(aq, m0, k0, 0, VB, fd, fs_t);
    warp_mma(ar, m0, k0, 0, VB, ff, fs_t);
    warp_mma(ac, m0, k0, 0, VB, [&](int m, int k) { return pair(s.x + m * LDX + k); },
                           [&](int k, int n) { return pair(s.e + n * LDS + k); });
  }
  __syncthreads();
  // dP and E take the places of P and T
  diagonal(ap, a.scale, s.diag, m0, p0);
  fade_scores<true, false>(ap, s.gates, m0, p0);
  fade_scores<true, false>(ae, s.gates, m0, p0);
  each_pair(ap, m0, p0, [&](int i, int j, float x, float y) {
    *reinterpret_cast<float2*>(s.p + i * LDP + j) = make_float2(a.scale * x, a.scale * y);
  });
  each_pair(ae, m0, p0, [&](int i, int j, float x, float y) {
    *reinterpret_cast<float2*>(s.t + i * LDP + j) = make_float2(x, y);
  });
  __syncthreads();
  auto fk_tok = [&](int k, int n) { return column<LDK>(sk + k * LDK + n); };
  const int i0 = m0 + (lane >> 2);
  float rl[2] = {0.f, 0.f}, rq[2] = {0.f, 0.f}, rr[2] = {0.f, 0.f}, rc[2] = {0.f, 0.f}, rg[2] = {0.f, 0.f};
  // sums over an accumulator's columns of tile * accumulator, per row
  auto row_dot = [&](float (&acc)[1][NK][4], const TI* tile, float (&out)[2]) {
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int c = k0 + 8 * j + 2 * (lane & 3);
      out[0] += acc[0][j][0] * ldf(tile + i0 * LDK + c) + acc[0][j][1] * ldf(tile + i0 * LDK + c + 1);
      out[1] += acc[0][j][2] * ldf(tile + (i0 + 8) * LDK + c) + acc[0][j][3] * ldf(tile + (i0 + 8) * LDK + c + 1);
    }
  };
  {
    float ag[1][NK][4];
    zero(ag);
    warp_mma(ag, m0, k0, 0, m0 + 16, [&](int m, int k) { return pair(s.t + m * LDP + k); }, fk_tok);
    row_dot(ag, sk, rg);
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + (r >= 2 ? 8 : 0);
        const float b = s.gates.beta[i], e = s.gates.start[i];
        ar[0][j][r] = -b * fmaf(e, ar[0][j][r], ag[0][j][r]);
        aq[0][j][r] *= a.scale * e;
        ac[0][j][r] *= s.gates.left[i];
      }
  }
  row_dot(ar, sk, rr);
  row_dot(ac, sk, rl);
#pragma unroll
  for (int j = 0; j < NK; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) ac[0][j][r] += ar[0][j][r];
  warp_mma(aq, m0, k0, 0, m0 + 16, [&](int m, int k) { return pair(s.p + m * LDP + k); }, fk_tok);
  row_dot(aq, sq, rq);
  // acc += dP_ii times row i of a tile
  auto add_diagonal = [&](float (&acc)[1][NK][4], const TI* tile) {
    const float d[2] = {s.diag[i0], s.diag[i0 + 8]};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[0][j][r] = fmaf(d[r >> 1], ldf(tile + (i0 + 8 * (r >> 1)) * LDK + k0 + 8 * j + 2 * (lane & 3) + (r & 1)), acc[0][j][r]);
  };
  add_diagonal(aq, sk);
  const size_t qo = dqk ? ((size_t)t0 * a.HV + hv) * a.K : qk, qstride = (size_t)(dqk ? a.HV : a.H) * a.K;
  auto put = [&](size_t at, int c, float x, float y, TI* out, float* part) {
    if (part) {
      if (c < a.K) part[at] = x;
      if (c + 1 < a.K) part[at + 1] = y;
    } else {
      if (c < a.K) stf(out + at, x);
      if (c + 1 < a.K) stf(out + at + 1, y);
    }
  };
  each_pair(aq, m0, k0, [&](int i, int c, float x, float y) {
    if (i < rows) put(qo + i * qstride + c, c, x, y, dq, dqk);
  });
  zero(aq);  // dk[column] without the terms with D
  warp_mma(aq, m0, k0, m0, BT, [&](int m, int k) { return column<LDP>(s.p + k * LDP + m); },
                       [&](int k, int n) { return column<LDK>(sq + k * LDK + n); });
  warp_mma(aq, m0, k0, m0, BT,
                         [&](int m, int k) {
                           const float2 x = column<LDP>(s.t + k * LDP + m), b = pair(s.gates.beta + k);
                           return make_float2(-b.x * x.x, -b.y * x.y);
                         },
                         fk_tok);
  row_dot(aq, sk, rc);
#pragma unroll
  for (int j = 0; j < NK; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) ac[0][j][r] += aq[0][j][r];
  add_diagonal(ac, sq);
  each_pair(ac, m0, k0, [&](int i, int c, float x, float y) {
    if (i < rows) put(qo + i * qstride + c, c, x, y, dk, dqk ? dqk + TK : nullptr);
  });
  // rows: over the four lanes of a row, then over the two warps that share it
  auto reduce = [&](float (&x)[2], int slot) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float y = x[r];
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      if ((lane & 3) == 0) s.red[slot][half][i0 + 8 * r] = y;
    }
  };
  reduce(rb, 0);
  reduce(rg, 1);
  reduce(rq, 2);
  reduce(rr, 3);
  reduce(rc, 4);
  reduce(rl, 5);
#pragma unroll
  for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
  if (lane == 0) s.dots[warp] = dot;
  __syncthreads();
  if (warp) return;
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) all += s.dots[w];
  float rc2[2], left[2], dg2[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = 2 * lane + r;
    auto row = [&](int slot) { return s.red[slot][0][i] + s.red[slot][1][i]; };
    rc2[r] = row(2) + row(3) - row(4);
    left[r] = row(5);
    if (i < rows) st_any(dbeta, a.dt_b, (size_t)(t0 + i) * a.HV + hv, row(0) - row(1));
  }
  gate_sums(rc2, left, s.gates.whole * all, dg2);
  const size_t at = (size_t)(t0 + 2 * lane) * a.HV + hv;
  if (2 * lane < rows) st_any(dg, a.dt_g, at, dg2[0]);
  if (2 * lane + 1 < rows) st_any(dg, a.dt_g, at + a.HV, dg2[1]);
}

template <int KP>
__global__ void __launch_bounds__(THREADS, sizeof(BwdSmem<KP>) <= 113 * 1024 ? 2 : 1)
    backward_kernel(Args a, const longlong2* __restrict__ tab, int VP, const float* __restrict__ tinv,
                    const float* __restrict__ states, const float* __restrict__ ds, const TI* __restrict__ dout,
                    TI* __restrict__ dq, TI* __restrict__ dk, TI* __restrict__ dv, void* __restrict__ dg,
                    void* __restrict__ dbeta, float* __restrict__ dqk) {
  griddep_launch_dependents();
  griddep_wait();
  backward_chunk<KP>(a, tab, VP, tinv, states, ds, dout, dq, dk, dv, dg, dbeta, dqk);
  zero_gradients(a, dq, dk, dv, dg, dbeta, dqk);
}

// dq, dk [T, H, K] = sums over the value heads of a key head, in their order.  One warp a row of K.
template <class TO>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* __restrict__ dqk, int64_t TH, int R, int K,
                                                        bool vec, TO* __restrict__ dq,
                                                        TO* __restrict__ dk) {
  griddep_launch_dependents();
  griddep_wait();
  const float* p = dqk + (blockIdx.y ? (size_t)TH * R * K : 0);
  TO* out = blockIdx.y ? dk : dq;
  const int lane = threadIdx.x & 31;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < TH; row += (int64_t)gridDim.x * 8) {
    const float* src = p + (size_t)row * R * K;
    if (vec) {
      for (int c = lane * 4; c < K; c += 128) {
        float4 x = *reinterpret_cast<const float4*>(src + c);
        for (int r = 1; r < R; ++r) {
          const float4 y = *reinterpret_cast<const float4*>(src + (size_t)r * K + c);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        const float v[4] = {x.x, x.y, x.z, x.w};
        Vec<TO, 4>::store(out + (size_t)row * K + c, v);
      }
    } else {
      for (int c = lane; c < K; c += 32) {
        float x = src[c];
        for (int r = 1; r < R; ++r) x += src[(size_t)r * K + c];
        stf(out + (size_t)row * K + c, x);
      }
    }
  }
}

template <int KP>
int adjoint32(const Args& a, const Saved& sv, int VP, const void* dout, float* inc, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(AdjSmem<KP>);
  allow_smem<adjoint_kernel<KP>>((int)smem);
  launch_pdl(adjoint_kernel<KP>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, sv.tinv, (const TI*)dout, inc);
  SSLA_CHECK_LAUNCH("gated_delta_rule adjoint");
  return SSLA_OK;
}

template <int KP>
int backward32(const Args& a, const Saved& sv, int VP, const float* ds, const Grads& g, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(BwdSmem<KP>);
  allow_smem<backward_kernel<KP>>((int)smem);
  launch_pdl(backward_kernel<KP>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, sv.tinv, sv.s, ds, (const TI*)g.dout,
                                                             (TI*)g.dq, (TI*)g.dk, (TI*)g.dv, g.dg, g.dbeta, g.dqk);
  SSLA_CHECK_LAUNCH("gated_delta_rule backward");
  return SSLA_OK;
}

template <class TO> int sum_heads(const Args& a, const Grads& g, cudaStream_t st) {
  const int64_t blocks = (a.T * a.H + 7) / 8;
  const bool vec = a.K % 4 == 0 && aligned_to(g.dq, 4 * sizeof(TO)) && aligned_to(g.dk, 4 * sizeof(TO));
  launch_pdl(sum_heads_kernel<TO>, dim3((unsigned)(blocks < 16 * kNumSMs ? blocks : 16 * kNumSMs), 2), dim3(256), 0, st, g.dqk, a.T * a.H, a.R, a.K, vec, (TO*)g.dq, (TO*)g.dk);
  SSLA_CHECK_LAUNCH("gated_delta_rule sum_heads");
  return SSLA_OK;
}

}  // namespace
}  // namespace delta
}  // namespace ssla

using namespace ssla;
using namespace ssla::delta;

extern "C" int ssla_chunk_gated_delta_rule_bwd(const void* q, const void* k, const void* v, const void* g,
                                               const void* beta, int dtype, int dtype_g, int dtype_beta,
                                               const int64_t* cu_seqlens, int64_t n_seqs, int64_t T, int64_t H,
                                               int64_t HV, int64_t K, int64_t V, float scale, int has_h0, int has_ht,
                                               const void* states, size_t states_bytes, const void* dout, const float* dht, void* dq,
                                               void* dk, void* dv, void* dg, void* dbeta, float* dh0, void* workspace,
                                               size_t workspace_bytes, ssla_stream_t stream) {
  const char* name = "ssla_chunk_gated_delta_rule_bwd";
  int rc = check_args(name, dtype, dtype_g, dtype_beta, n_seqs, T, H, HV, K, V);
  if (rc) return rc;
  if (HV == 0) return SSLA_OK;
  SSLA_CHECK_ARG(cu_seqlens && states, "%s: null pointer", name);
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && dout && dq && dk && dv && dg && dbeta), "%s: null pointer", name);
  const bool exact = exact_states(dtype, has_h0, has_ht);  // as in the forward
  SSLA_CHECK_ARG(!dh0 || has_h0, "%s: dh0 without an initial state", name);
  const Plan p = make_plan(n_seqs, T, HV, K, V);
  const int KP = pad_k(K), VP = pad_v(V);
  Saved sv;
  Work w;
  const size_t need = saved_layout(const_cast<void*>(states), p, dtype, exact, n_seqs, HV, KP, VP, &sv);
  const size_t need_w = work_layout(workspace, p, T, H, HV, K, KP, VP, true, &w);
  if (states_bytes < need || workspace_bytes < need_w || (need_w && !workspace)) {
    set_error("%s: states of %zu bytes and workspace of %zu, %zu and %zu needed", name, states_bytes, workspace_bytes,
              need, need_w);
    return SSLA_ERR_WORKSPACE;
  }
  SSLA_CHECK_ARG(aligned_to(states, 16) && aligned_to(workspace, 16), "%s: states and workspace must be 16-byte aligned", name);
  cudaStream_t st = (cudaStream_t)stream;
  const Args a = make_args(q, k, v, g, beta, dtype, dtype_g, dtype_beta, cu_seqlens, n_seqs, T, H, HV, K, V, scale);
  const int64_t items = p.MC * HV, blocks = items > 0 ? items : 1;
  const bool f32 = dtype == SSLA_F32;
  if (items > 0) {
    rc = !f32       ? adjoint16(dtype, a, sv, KP, VP, t_planes(exact), dout, w.inc, items, st)
         : KP == 64 ? adjoint32<64>(a, sv, VP, dout, w.inc, items, st)
                    : adjoint32<128>(a, sv, VP, dout, w.inc, items, st);
    if (rc) return rc;
  }
  rc = run_chain(p, sv, w, w.ds, dht, dh0, n_seqs, (int)HV, (int)K, (int)V, true, exact, !f32, st);
  if (rc || T == 0) return rc;
  const Grads gr = {dout, dq, dk, dv, dg, dbeta, a.R > 1 ? w.dqk : nullptr};
  rc = !f32       ? backward16(dtype, a, sv, KP, VP, t_planes(exact), w.ds, gr, blocks, st)
       : KP == 64 ? backward32<64>(a, sv, VP, w.ds, gr, blocks, st)
                  : backward32<128>(a, sv, VP, w.ds, gr, blocks, st);
  if (rc || !gr.dqk) return rc;
  return SSLA_DISPATCH_DTYPE(dtype, T_, [&] { return sum_heads<T_>(a, gr, st); });
}
