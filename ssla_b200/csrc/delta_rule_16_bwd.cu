// Chunked gated delta rule for bf16 and fp16 tokens, backward: the kernels of delta_rule_bwd.cu on
// bf16 planes (formulas there, planes in delta_rule_16.cuh).
#include "delta_rule_16.cuh"

namespace ssla {
namespace delta {
namespace {

using namespace h16;

// ------------------------------------------------------------------ adjoint of the chunk maps
template <class TI, int KP, int NI> struct Adj16 {
  static constexpr int N = Planes<TI>::n, LDK = KP + 8;
  bf k[N * BT * LDK];
  bf q[N * BT * LDK];
  bf d[N * BT * LDT];
  bf t[NI * FRAG_ELEMS];
  bf w[NI * BT * LDK];  // beta exp(gc) K, then W, then scale qh
  bf p[NI * BT * LDT];  // P; then every second panel of dO
  Gates gates;
};

template <class TI, int KP, int NI>
__global__ void __launch_bounds__(THREADS, sizeof(Adj16<TI, KP, NI>) <= 75 * 1024 ? 3 : sizeof(Adj16<TI, KP, NI>) <= 113 * 1024 ? 2 : 1)
    adjoint16_kernel(Args a, const longlong2* __restrict__ tab, int VP, const bf* __restrict__ tinv,
                     const TI* __restrict__ dout, float* __restrict__ inc) {
  griddep_launch_dependents();
  griddep_wait();
  using S = Adj16<TI, KP, NI>;
  constexpr int N = S::N, LDK = S::LDK, PLK = BT * LDK, PLT = BT * LDT, NK = KP / 16;
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
  load_tokens<TI, LDK, KP, THREADS>(s.k, (const TI*)a.k + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_tokens<TI, LDK, KP, THREADS>(s.q, (const TI*)a.q + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  copy16<THREADS>(s.t, tinv + item * (NI * FRAG_ELEMS), NI * FRAG_BYTES);
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V;
  const bool vec_d = a.vec_v && (reinterpret_cast<uintptr_t>(dout) & 15) == 0;
  auto load_d = [&](int v0) {
    load_tokens<TI, LDT, 64, THREADS>(v0 & 64 ? s.p : s.d, dout + vo + v0, (size_t)a.HV * a.V, rows, a.V - v0, vec_d);
    cp_commit();
  };
  load_d(0);
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  cp_wait<0>();
  __syncthreads();
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32, k0 = (warp & 1) * (KP / 2);
  {
    float acc[1][4][4];
    zero(acc);
    if (n0 <= m0) mm(acc, RowA<LDK, PLK, N>(s.q), ColB<LDK, PLK, N>(s.k), m0, n0, 0, KP);
    fade_scores<false, (NI < 3)>(acc, s.gates, m0, n0);
    each_pair(acc, m0, n0, [&](int i, int j, float x, float y) { put<NI, PLT>(s.p + i * LDT + j, x, y); });
  }
  for (int i = threadIdx.x; i < BT * KP / 2; i += THREADS) {
    const int r = i / (KP / 2), c = (i % (KP / 2)) * 2;
    float2 x = pair(s.k + r * LDK + c);
    if (N > 1) {
      const float2 y = pair(s.k + PLK * (N - 1) + r * LDK + c);
      x.x += y.x;
      x.y += y.y;
    }
    const float f = s.gates.beta[r] * s.gates.start[r];
    put<NI, PLK>(s.w + r * LDK + c, f * x.x, f * x.y);
  }
  __syncthreads();
  const RowB<LDK, PLK, NI> wb(s.w);
  float acc[1][NK][4];
  zero(acc);
  mm(acc, FragA<NI, false>(s.t), wb, m0, k0, 0, m0 + 16);
  __syncthreads();
  each_pair(acc, m0, k0, [&](int i, int n, float x, float y) { put<NI, PLK>(s.w + i * LDK + n, x, y); });
  __syncthreads();
  zero(acc);
  mm(acc, RowA<LDT, PLT, NI>(s.p), wb, m0, k0, 0, m0 + 16);
  __syncthreads();
  const int i0 = m0 + ((threadIdx.x & 31) >> 2);
  const float e0 = s.gates.start[i0], e1 = s.gates.start[i0 + 8];
  each_pair(acc, m0, k0, [&](int i, int n, float& x, float& y) {
    float2 z = pair(s.q + i * LDK + n);
    if (N > 1) {
      const float2 y2 = pair(s.q + PLK * (N - 1) + i * LDK + n);
      z.x += y2.x;
      z.y += y2.y;
    }
    const float e = i == i0 ? e0 : e1;
    x = a.scale * (e * z.x - x);
    y = a.scale * (e * z.y - y);
  });
  each_pair(acc, m0, k0, [&](int i, int n, float x, float y) { put<NI, PLK>(s.w + i * LDK + n, x, y); });
  constexpr int MT = KP / 64;
  const int mk = (warp >> 1) * 16 * MT;
  for (int v0 = 0; v0 < VP; v0 += 64) {
    cp_wait<0>();
    __syncthreads();  // this panel is there, the other place is read
    if (v0 + 64 < VP) load_d(v0 + 64);
    float o[MT][4][4];
    zero(o);
    mm(o, ColA<LDK, PLK, NI>(s.w), RowB<LDT, PLT, N>(v0 & 64 ? s.p : s.d), mk, n0, 0, BT);
    each_pair(o, mk, n0, [&](int m, int n, float x, float y) {
      *reinterpret_cast<float2*>(inc_at(inc, item, KP, VP, m, v0 + n)) = make_float2(x, y);
    });
  }
}

// ------------------------------------------------------------------ gradients of a chunk
// Warps: 4 groups of 16 rows x CG column groups.
template <class TI, int KP> struct Bwd16 {
  static constexpr int N = Planes<TI>::n, LDK = KP + 8, VB = N > 1 ? 32 : KP / 2, LDX = VB + 8, CG = VB / 16, NTH = 128 * CG;
  bf k[N * BT * LDK];
  bf q[N * BT * LDK];
  bf d[N * BT * LDX];
  bf t[2 * FRAG_ELEMS];
  bf p[2 * BT * LDT];  // P, then dP below its diagonal
  bf x[2 * BT * LDX];  // beta X, then U;  x and f at last -beta E
  bf f[2 * BT * LDX];  // dU, then F
  bf s[2 * KP * LDX];  // S;  s and e at last E
  bf e[2 * KP * LDX];  // D
  float red[6][CG][BT];
  float dots[NTH / 32];
  float diag[BT];  // of dP
  Gates gates;
  static_assert(4 * BT * LDX >= 2 * BT * LDT && 4 * KP * LDX >= 2 * BT * LDT, "E fits the panels' places");
};

template <class TI, int KP>
__device__ __forceinline__ void backward16_chunk(const Args& a, const longlong2* __restrict__ tab, int VP, int tplanes,
                                                 const bf* __restrict__ tinv, const bf* __restrict__ states,
                                                 const bf* __restrict__ ds, const TI* __restrict__ dout,
                                                 TI* __restrict__ dq, TI* __restrict__ dk, TI* __restrict__ dv,
                                                 void* __restrict__ dg, void* __restrict__ dbeta,
                                                 float* __restrict__ dqk) {
  using S = Bwd16<TI, KP>;
  constexpr int N = S::N, LDK = S::LDK, VB = S::VB, LDX = S::LDX, CG = S::CG, NTH = S::NTH;
  constexpr int PLK = BT * LDK, PLX = BT * LDX, PLT = BT * LDT, PLS = KP * LDX;
  constexpr int NT = VB / CG / 8, NK = KP / CG / 8, NP = BT / CG / 8;  // tiles of a warp's columns
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
  load_tokens<TI, LDK, KP, NTH>(s.k, (const TI*)a.k + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_tokens<TI, LDK, KP, NTH>(s.q, (const TI*)a.q + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  const int cg = warp & (CG - 1), m0 = (warp / CG) * 16, i0 = m0 + (lane >> 2);
  const int n0 = cg * (VB / CG), p0 = cg * (BT / CG), k0 = cg * (KP / CG);
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V, vstride = (size_t)a.HV * a.V;
  const bool vec_d = a.vec_v && (reinterpret_cast<uintptr_t>(dout) & 15) == 0;
  const bool even = a.V % 2 == 0 && reinterpret_cast<uintptr_t>(a.v) % 4 == 0;
  const int width_v = store_width(dv, a.V);
  const TI* gv = (const TI*)a.v + vo;
  copy16<NTH>(s.t, tinv + item * ((size_t)tplanes * FRAG_ELEMS), 2 * FRAG_BYTES);
  const FragA<2, false> t_a(s.t);
  const FragA<2, true> tt_a(s.t);
  const bf* gs = states + item * (2 * KP * VP);
  const bf* ge = ds + item * (2 * KP * VP);
  const RowA<LDK, PLK, N> k_a(s.k), q_a(s.q);
  const RowB<LDK, PLK, N> k_b(s.k), q_b(s.q);
  const RowB<LDX, PLX, 2> x_b(s.x), f_b(s.f);
  const RowB<LDX, PLX, N> d_b(s.d);
  const RowA<LDX, PLX, N> d_a(s.d);
  const RowA<LDX, PLX, 2> x_a(s.x), f_a(s.f);
  const ColB<LDX, PLX, 2> x_t(s.x);
  const ColB<LDX, PLS, 2> s_t(s.s), e_t(s.e);
  const RowB<LDX, PLS, 2> s_b(s.s), e_b(s.e);
  const ColA<LDT, PLT, 2> p_t(s.p);

  float aq[1][NK][4], ar[1][NK][4], ac[1][NK][4];  // dO S^T, F S^T, U D^T
  float ap[1][NP][4], ae[1][NP][4];                // dO U^T, F U^T
  zero(aq); zero(ar); zero(ac); zero(ap); zero(ae);
  float rb[2] = {0.f, 0.f}, dot = 0.f;
  const bool low = p0 <= m0 + 15;
  for (int v0 = 0; v0 < a.V; v0 += VB) {
    __syncthreads();
    load_planes<LDX, KP, VB, NTH>(s.s, gs + v0, VP);
    load_planes<LDX, KP, VB, NTH>(s.e, ge + v0, VP);
    load_tokens<TI, LDX, VB, NTH>(s.d, dout + vo + v0, vstride, rows, a.V - v0, vec_d);
    cp_commit();
    if (v0 == 0) {
      cp_wait<1>();
      __syncthreads();
      float acc[1][NP][4];
      zero(acc);
      if (low) mm(acc, q_a, ColB<LDK, PLK, N>(s.k), m0, p0, 0, KP);
      fade_scores<false, true>(acc, s.gates, m0, p0);
      each_pair(acc, m0, p0, [&](int i, int j, float x, float y) { put<2, PLT>(s.p + i * LDT + j, x, y); });
    }
    float xv[1][NT][4];
    load_pairs(xv, gv + v0, vstride, rows, a.V - v0, m0, n0, even);
    cp_wait<0>();
    __syncthreads();
    float ks[1][NT][4], du[1][NT][4];
    zero(ks);
    zero(du);
    mm_ab_ac(ks, s_b, du, e_b, k_a, m0, n0, 0, KP);
    const float be[2] = {s.gates.beta[i0], s.gates.beta[i0 + 8]};
    const float ee[2] = {s.gates.start[i0], s.gates.start[i0 + 8]}, le[2] = {s.gates.left[i0], s.gates.left[i0 + 8]};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        xv[0][j][r] -= ee[r >> 1] * ks[0][j][r];
        du[0][j][r] *= le[r >> 1];
      }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        put<2, PLX>(s.x + (i0 + 8 * r) * LDX + n0 + 8 * j + 2 * (lane & 3), be[r] * xv[0][j][2 * r], be[r] * xv[0][j][2 * r + 1]);
    for (int i = tid; i < KP * (VB / 2); i += NTH) {
      const int at = (i / (VB / 2)) * LDX + (i % (VB / 2)) * 2;
      const float2 x0 = pair(s.s + at), x1 = pair(s.s + PLS + at), y0 = pair(s.e + at), y1 = pair(s.e + PLS + at);
      dot += (x0.x + x1.x) * (y0.x + y1.x) + (x0.y + x1.y) * (y0.y + y1.y);
    }
    __syncthreads();
    zero(ks);
    mm(ks, t_a, x_b, m0, n0, 0, m0 + 16);  // U
    {
      float pd[1][NT][4];
      zero(pd);
      mm(pd, p_t, d_b, m0, n0, m0, BT);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) du[0][j][r] = fmaf(a.scale, pd[0][j][r], du[0][j][r]);
    }
    __syncthreads();
    each_pair(ks, m0, n0, [&](int i, int n, float x, float y) { put<2, PLX>(s.x + i * LDX + n, x, y); });
    each_pair(du, m0, n0, [&](int i, int n, float x, float y) { put<2, PLX>(s.f + i * LDX + n, x, y); });
    __syncthreads();
    zero(du);
    mm(du, tt_a, f_b, m0, n0, m0, BT);  // F
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      rb[0] += du[0][j][0] * xv[0][j][0] + du[0][j][1] * xv[0][j][1];
      rb[1] += du[0][j][2] * xv[0][j][2] + du[0][j][3] * xv[0][j][3];
    }
    {
      float out[1][NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) out[0][j][r] = be[r >> 1] * du[0][j][r];
      store_rows(out, 1.f, dv + vo + v0, vstride, rows, a.V - v0, m0, n0, width_v);
    }
    __syncthreads();
    each_pair(du, m0, n0, [&](int i, int n, float x, float y) { put<2, PLX>(s.f + i * LDX + n, x, y); });
    __syncthreads();
    if (low) mm_ab_cb(ap, d_a, ae, f_a, x_t, m0, p0, 0, VB);
    mm_ab_cb(aq, d_a, ar, f_a, s_t, m0, k0, 0, VB);
    mm(ac, x_a, e_t, m0, k0, 0, VB);
  }
  __syncthreads();
  bf* const sE = s.s;  // E;  -beta E at s.x
  const float be[2] = {s.gates.beta[i0], s.gates.beta[i0 + 8]}, ee[2] = {s.gates.start[i0], s.gates.start[i0 + 8]};
  const float le[2] = {s.gates.left[i0], s.gates.left[i0 + 8]};
  diagonal(ap, a.scale, s.diag, m0, p0);
  fade_scores<true, true>(ap, s.gates, m0, p0);
  fade_scores<true, true>(ae, s.gates, m0, p0);
  each_pair(ap, m0, p0, [&](int i, int j, float x, float y) { put<2, PLT>(s.p + i * LDT + j, a.scale * x, a.scale * y); });
  each_pair(ae, m0, p0, [&](int i, int j, float x, float y) {
    put<2, PLT>(sE + i * LDT + j, x, y);
    const float b = i == i0 ? -be[0] : -be[1];
    put<2, PLT>(s.x + i * LDT + j, b * x, b * y);
  });
  __syncthreads();
  float rl[2] = {0.f, 0.f}, rq[2] = {0.f, 0.f}, rr[2] = {0.f, 0.f}, rc[2] = {0.f, 0.f}, rg[2] = {0.f, 0.f};
  auto token_pair = [&](const bf* tile, int j, int r) {
    const bf* p = tile + (i0 + 8 * r) * LDK + k0 + 8 * j + 2 * (lane & 3);
    float2 z = pair(p);
    if (N > 1) {
      const float2 y = pair(p + (N - 1) * PLK);
      z.x += y.x;
      z.y += y.y;
    }
    return z;
  };
  auto row_dot = [&](float (&acc)[1][NK][4], const bf* tile, float (&out)[2]) {
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 z = token_pair(tile, j, r);
        out[r] += acc[0][j][2 * r] * z.x + acc[0][j][2 * r + 1] * z.y;
      }
  };
  // acc += dP_ii times row i of a tile
  auto add_diagonal = [&](float (&acc)[1][NK][4], const bf* tile) {
    const float d[2] = {s.diag[i0], s.diag[i0 + 8]};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float2 z = token_pair(tile, j, r);
        acc[0][j][2 * r] = fmaf(d[r], z.x, acc[0][j][2 * r]);
        acc[0][j][2 * r + 1] = fmaf(d[r], z.y, acc[0][j][2 * r + 1]);
      }
  };
  {
    float ag[1][NK][4];
    zero(ag);
    mm(ag, RowA<LDT, PLT, 2>(sE), k_b, m0, k0, 0, m0 + 16);
    row_dot(ag, s.k, rg);
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ar[0][j][r] = -be[r >> 1] * fmaf(ee[r >> 1], ar[0][j][r], ag[0][j][r]);
        aq[0][j][r] *= a.scale * ee[r >> 1];
        ac[0][j][r] *= le[r >> 1];
      }
  }
  row_dot(ar, s.k, rr);
  row_dot(ac, s.k, rl);
#pragma unroll
  for (int j = 0; j < NK; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) ac[0][j][r] += ar[0][j][r];
  mm(aq, RowA<LDT, PLT, 2>(s.p), k_b, m0, k0, 0, m0 + 16);
  row_dot(aq, s.q, rq);
  add_diagonal(aq, s.k);
  const size_t qo = dqk ? ((size_t)t0 * a.HV + hv) * a.K : qk, qstride = (size_t)(dqk ? a.HV : a.H) * a.K;
  auto write = [&](float (&acc)[1][NK][4], TI* out, float* part) {
    if (!part) {
      store_rows(acc, 1.f, out + qo, qstride, rows, a.K, m0, k0, store_width(out, a.K));
      return;
    }
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = i0 + 8 * r, c = k0 + 8 * j + 2 * (lane & 3);
        if (i >= rows || c >= a.K) continue;
        const float x = acc[0][j][2 * r], y = acc[0][j][2 * r + 1];
        float* const p = part + qo + i * qstride + c;
        if (a.K % 2 == 0) {
          *reinterpret_cast<float2*>(p) = make_float2(x, y);
        } else {
          p[0] = x;
          if (c + 1 < a.K) p[1] = y;
        }
      }
  };
  write(aq, dq, dqk);
  zero(aq);  // dk[column] without the terms with D
  mm(aq, p_t, q_b, m0, k0, m0, BT);
  mm(aq, ColA<LDT, PLT, 2>(s.x), k_b, m0, k0, m0, BT);
  row_dot(aq, s.k, rc);
#pragma unroll
  for (int j = 0; j < NK; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) ac[0][j][r] += aq[0][j][r];
  add_diagonal(ac, s.q);
  write(ac, dk, dqk ? dqk + TK : nullptr);
  auto reduce = [&](float (&x)[2], int slot) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float y = x[r];
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      if ((lane & 3) == 0) s.red[slot][cg][i0 + 8 * r] = y;
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
  for (int w = 0; w < NTH / 32; ++w) all += s.dots[w];
  float rc2[2], left[2], dg2[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = 2 * lane + r;
    auto row = [&](int slot) {
      float x = 0.f;
#pragma unroll
      for (int c = 0; c < CG; ++c) x += s.red[slot][c][i];
      return x;
    };
    rc2[r] = row(2) + row(3) - row(4);
    left[r] = row(5);
    if (i < rows) st_any(dbeta, a.dt_b, (size_t)(t0 + i) * a.HV + hv, row(0) - row(1));
  }
  gate_sums(rc2, left, s.gates.whole * all, dg2);
  const size_t at = (size_t)(t0 + 2 * lane) * a.HV + hv;
  if (2 * lane < rows) st_any(dg, a.dt_g, at, dg2[0]);
  if (2 * lane + 1 < rows) st_any(dg, a.dt_g, at + a.HV, dg2[1]);
}

template <class TI, int KP>
__global__ void __launch_bounds__(Bwd16<TI, KP>::NTH, sizeof(Bwd16<TI, KP>) <= 113 * 1024 ? 2 : 1)
    backward16_kernel(Args a, const longlong2* __restrict__ tab, int VP, int tplanes, const bf* __restrict__ tinv,
                      const bf* __restrict__ states, const bf* __restrict__ ds, const TI* __restrict__ dout,
                      TI* __restrict__ dq, TI* __restrict__ dk, TI* __restrict__ dv, void* __restrict__ dg,
                      void* __restrict__ dbeta, float* __restrict__ dqk) {
  griddep_launch_dependents();
  griddep_wait();
  backward16_chunk<TI, KP>(a, tab, VP, tplanes, tinv, states, ds, dout, dq, dk, dv, dg, dbeta, dqk);
  zero_gradients(a, dq, dk, dv, dg, dbeta, dqk);
}

template <class TI, int KP, int NI>
int adjoint(const Args& a, const Saved& sv, int VP, const void* dout, float* inc, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(Adj16<TI, KP, NI>);
  allow_smem<adjoint16_kernel<TI, KP, NI>>((int)smem);
  launch_pdl(adjoint16_kernel<TI, KP, NI>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, (const bf*)sv.tinv,
                                                                      (const TI*)dout, inc);
  SSLA_CHECK_LAUNCH("gated_delta_rule adjoint");
  return SSLA_OK;
}

template <class TI, int KP>
int backward(const Args& a, const Saved& sv, int VP, int tplanes, const bf* ds, const Grads& g, int64_t items,
             cudaStream_t st) {
  const size_t smem = sizeof(Bwd16<TI, KP>);
  allow_smem<backward16_kernel<TI, KP>>((int)smem);
  launch_pdl(backward16_kernel<TI, KP>, dim3((unsigned)items), dim3(Bwd16<TI, KP>::NTH), smem, st, a, sv.chunk_tab, VP, tplanes, (const bf*)sv.tinv, (const bf*)sv.s, ds, (const TI*)g.dout, (TI*)g.dq, (TI*)g.dk,
      (TI*)g.dv, g.dg, g.dbeta, g.dqk);
  SSLA_CHECK_LAUNCH("gated_delta_rule backward");
  return SSLA_OK;
}

}  // namespace

int adjoint16(int dtype, const Args& a, const Saved& sv, int KP, int VP, int planes, const void* dout, float* inc,
              int64_t items, cudaStream_t st) {
  if (dtype == SSLA_F16)
    return KP == 64 ? adjoint<__half, 64, 3>(a, sv, VP, dout, inc, items, st)
                    : adjoint<__half, 128, 3>(a, sv, VP, dout, inc, items, st);
  if (planes == 3)
    return KP == 64 ? adjoint<bf, 64, 3>(a, sv, VP, dout, inc, items, st) : adjoint<bf, 128, 3>(a, sv, VP, dout, inc, items, st);
  return KP == 64 ? adjoint<bf, 64, 2>(a, sv, VP, dout, inc, items, st) : adjoint<bf, 128, 2>(a, sv, VP, dout, inc, items, st);
}

int backward16(int dtype, const Args& a, const Saved& sv, int KP, int VP, int planes, const void* ds, const Grads& g,
               int64_t items, cudaStream_t st) {
  const bf* d = (const bf*)ds;
  if (dtype == SSLA_F16)
    return KP == 64 ? backward<__half, 64>(a, sv, VP, planes, d, g, items, st)
                    : backward<__half, 128>(a, sv, VP, planes, d, g, items, st);
  return KP == 64 ? backward<bf, 64>(a, sv, VP, planes, d, g, items, st) : backward<bf, 128>(a, sv, VP, planes, d, g, items, st);
}

}  // namespace delta
}  // namespace ssla
