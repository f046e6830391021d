// Chunked gated delta rule for bf16 and fp16 tokens: prep and output kernels on bf16 planes
// (delta_rule_16.cuh; the formulas are in delta_rule.cuh).  The chain between them is delta_rule.cu's.
#include "delta_rule_16.cuh"
#include "delta_rule_inverse.cuh"

namespace ssla {
namespace delta {
namespace {

using namespace h16;

// ------------------------------------------------------------------ prep
// NI planes of intermediate results: 3 where the states leave in fp32, else 2.
template <class TI, int KP, int NI> struct Prep16 {
  static constexpr int NT = Planes<TI>::n, LDK = KP + 8;
  bf k[NT * BT * LDK];
  bf v[NT * BT * LDT];
  union {
    float a[BT * LDC];     // A; once inverted
    bf tc[NI * BT * LDT];  // planes of T diag(..)
  };
  float t[BT * LDC];
  bf y[(NI > 2 ? NI : 2) * BT * LDT];  // scratch of the inverse, then planes of a panel
  unsigned red[THREADS / 32];
  Gates gates;
};

// Planes of T as fragments.
template <int NI> __device__ __forceinline__ void write_t(const float* t, bf* out) {
  for (int f = threadIdx.x; f < FRAGS; f += THREADS) {
    const int lane = f & 31, blk = f >> 5;
    const int mb = blk >= 6 ? 3 : blk >= 3 ? 2 : blk >= 1 ? 1 : 0, kb = blk - mb * (mb + 1) / 2;
    const float* p = t + (16 * mb + (lane >> 2)) * LDC + 16 * kb + 2 * (lane & 3);
    uint32_t w[NI][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 x = pair(p + (j & 1) * 8 * LDC + (j >> 1) * 8);
#pragma unroll
      for (int q = 0; q < NI; ++q) {
        w[q][j] = pack(x.x, x.y);
        rest(w[q][j], x.x, x.y);
      }
    }
#pragma unroll
    for (int q = 0; q < NI; ++q)
      reinterpret_cast<uint4*>(out)[q * FRAGS + f] = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
}

template <class TI, int KP, int NI>
__global__ void __launch_bounds__(THREADS, sizeof(Prep16<TI, KP, NI>) <= 75 * 1024 ? 3 : sizeof(Prep16<TI, KP, NI>) <= 113 * 1024 ? 2 : 1)
    prep16_kernel(Args a, const longlong2* __restrict__ tab, int VP, bf* __restrict__ tinv, unsigned char* __restrict__ pm,
                  float* __restrict__ inc) {
  griddep_launch_dependents();
  griddep_wait();
  using S = Prep16<TI, KP, NI>;
  constexpr int N = S::NT, LDK = S::LDK, PLK = BT * LDK, PLT = BT * LDT;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
  constexpr int NPL = pm_planes(NI > 2);
  unsigned char* const record = pm + item * pm_bytes(KP, NPL);
  const int warp = threadIdx.x >> 5;
  load_tokens<TI, LDK, KP, THREADS>(s.k, (const TI*)a.k + ((size_t)t0 * a.H + h) * a.K, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  auto load_v = [&](int v0) {
    load_tokens<TI, LDT, 64, THREADS>(s.v, (const TI*)a.v + ((size_t)t0 * a.HV + hv) * a.V + v0, (size_t)a.HV * a.V,
                                      rows, a.V - v0, a.vec_v);
    cp_commit();
  };
  load_v(0);
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  cp_wait<0>();
  __syncthreads();
  if (threadIdx.x == 0) *reinterpret_cast<float*>(record) = s.gates.whole;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  {
    float acc[1][4][4];
    zero(acc);
    if (n0 <= m0) mm(acc, RowA<LDK, PLK, N>(s.k), ColB<LDK, PLK, N>(s.k), m0, n0, 0, KP);
    fade_scores<true, (NI < 3)>(acc, s.gates, m0, n0);
    const int i0 = m0 + ((threadIdx.x & 31) >> 2);
    const float b0 = s.gates.beta[i0], b1 = s.gates.beta[i0 + 8];
    each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
      const float b = i == i0 ? b0 : b1;
      *reinterpret_cast<float2*>(s.a + i * LDC + j) = make_float2(b * x, b * y);
    });
  }
  __syncthreads();
  unit_lower_inverse(s.a, s.t, reinterpret_cast<float*>(s.y));
  write_t<NI>(s.t, tinv + item * (NI * FRAG_ELEMS));
  auto scale_t = [&](bool w) {  // tc = T diag(beta [exp(gc)])
    for (int i = threadIdx.x; i < BT * BT / 2; i += THREADS) {
      const int r = i >> 5, c = (i & 31) * 2;
      const float2 x = pair(s.t + r * LDC + c), b = pair(s.gates.beta + c), e = pair(s.gates.start + c);
      put<NI, PLT>(s.tc + r * LDT + c, x.x * b.x * (w ? e.x : 1.f), x.y * b.y * (w ? e.y : 1.f));
    }
  };
  scale_t(true);
  __syncthreads();
  const int panels = KP / 64 + VP / 64;
  for (int p = 0; p < panels; ++p) {
    const bool w = p < KP / 64;
    const int c0 = (w ? p : p - KP / 64) * 64;
    {
      float acc[1][4][4];
      zero(acc);
      const RowA<LDT, PLT, NI> t(s.tc);
      if (w) mm(acc, t, RowB<LDK, PLK, N>(s.k + c0), m0, n0, 0, m0 + 16);
      else mm(acc, t, RowB<LDT, PLT, N>(s.v), m0, n0, 0, m0 + 16);
      const int i0 = m0 + ((threadIdx.x & 31) >> 2);
      const float l0 = s.gates.left[i0], l1 = s.gates.left[i0 + 8];
      each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
        const float l = i == i0 ? l0 : l1;
        put<NI, PLT>(s.y + i * LDT + j, x * l, y * l);
      });
    }
    __syncthreads();
    if (p + 1 == KP / 64) scale_t(false);  // tc and v are read: the next panel's
    if (!w && c0 + 64 < VP) load_v(c0 + 64);
    {
      constexpr int MT = KP / 64;
      float acc[MT][4][4];
      zero(acc);
      const int mk = (warp >> 1) * 16 * MT;
      mm(acc, ColA<LDK, PLK, N>(s.k), RowB<LDT, PLT, NI>(s.y), mk, n0, 0, BT);
      if (w)
        store_pm<KP, NPL>(acc, mk, c0, n0, s.red, record);
      else
        each_pair(acc, mk, n0, [&](int m, int n, float x, float y) {
          *reinterpret_cast<float2*>(inc_at(inc, item, KP, VP, m, c0 + n)) = make_float2(x, y);
        });
    }
    cp_wait<0>();
    __syncthreads();  // the readers of y are done
  }
}

// ------------------------------------------------------------------ output
// 4 row groups of 16 x 2 column groups of warps, panels of 64 value columns.  X and U take the place
// of the state's panel, so that two blocks (K = 128; three at K = 64) fit an SM: 224 us for the 32768-token
// prompt of 8 heads, 22 us less than with panels of 32 columns.  One block of 16 warps with places of their
// own was slower than either (340 us).
template <class TI, int KP> struct Out16 {
  static constexpr int N = Planes<TI>::n, LDK = KP + 8, VB = 64, LDX = VB + 8, CG = 2, NTH = 128 * CG;
  bf k[N * BT * LDK];
  bf q[N * BT * LDK];
  bf t[2 * FRAG_ELEMS];
  bf p[2 * BT * LDT];
  bf s[2 * KP * LDX];  // S, then beta X, then U
  Gates gates;
  static constexpr int resident(size_t bytes) { return bytes <= 75 * 1024 ? 3 : bytes <= 113 * 1024 ? 2 : 1; }
};

template <class TI, int KP>
__device__ __forceinline__ void output16_chunk(const Args& a, const longlong2* __restrict__ tab, int VP, int tplanes,
                                               const bf* __restrict__ tinv, const bf* __restrict__ states,
                                               TI* __restrict__ o) {
  using S = Out16<TI, KP>;
  constexpr int N = S::N, LDK = S::LDK, CG = S::CG, NTH = S::NTH, PLK = BT * LDK, PLT = BT * LDT, VB = S::VB, LDX = S::LDX, PLX = BT * LDX, NT = VB / CG / 8, NP = 8 / CG;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cg = warp & (CG - 1), m0 = (warp / CG) * 16, n0 = cg * (VB / CG), p0 = cg * (64 / CG), i0 = m0 + (lane >> 2);
  const size_t qk = ((size_t)t0 * a.H + h) * a.K;
  load_tokens<TI, LDK, KP, NTH>(s.k, (const TI*)a.k + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  load_tokens<TI, LDK, KP, NTH>(s.q, (const TI*)a.q + qk, (size_t)a.H * a.K, rows, a.K, a.vec_k);
  cp_commit();
  copy16<NTH>(s.t, tinv + item * ((size_t)tplanes * FRAG_ELEMS), 2 * FRAG_BYTES);
  const bf* st = states + item * (2 * KP * VP);
  load_planes<LDX, KP, VB, NTH>(s.s, st, VP);
  cp_commit();
  if (warp == 0) load_gates(s.gates, a, t0, rows, hv);
  cp_wait<1>();
  __syncthreads();
  {
    float acc[1][NP][4];
    zero(acc);
    if (p0 <= m0 + 15) mm(acc, RowA<LDK, PLK, N>(s.q), ColB<LDK, PLK, N>(s.k), m0, p0, 0, KP);
    fade_scores<false, true>(acc, s.gates, m0, p0);
    each_pair(acc, m0, p0, [&](int i, int j, float x, float y) { put<2, PLT>(s.p + i * LDT + j, x, y); });
  }
  const FragA<2, false> t_a(s.t);
  const RowB<LDX, KP * LDX, 2> s_b(s.s);
  bf* const sx = s.s;
  const RowB<LDX, PLX, 2> x_b(sx);
  const float be[2] = {s.gates.beta[i0], s.gates.beta[i0 + 8]};
  const float ee[2] = {s.gates.start[i0], s.gates.start[i0 + 8]};
  const size_t vo = ((size_t)t0 * a.HV + hv) * a.V, vstride = (size_t)a.HV * a.V;
  const TI* gv = (const TI*)a.v + vo;
  const bool even = a.V % 2 == 0 && reinterpret_cast<uintptr_t>(a.v) % 4 == 0;
  const int width = store_width(o, a.V);
  for (int v0 = 0; v0 < a.V; v0 += VB) {
    if (v0) {
      __syncthreads();  // readers of the previous panel are done
      load_planes<LDX, KP, VB, NTH>(s.s, st + v0, VP);
      cp_commit();
    }
    float xv[1][NT][4];
    load_pairs(xv, gv + v0, vstride, rows, a.V - v0, m0, n0, even);
    cp_wait<0>();
    __syncthreads();
    float aq[1][NT][4], ak[1][NT][4];
    zero(aq);
    zero(ak);
    mm_ab_cb(ak, RowA<LDK, PLK, N>(s.k), aq, RowA<LDK, PLK, N>(s.q), s_b, m0, n0, 0, KP);
    __syncthreads();  // S is read
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        put<2, PLX>(sx + (i0 + 8 * r) * LDX + n0 + 8 * j + 2 * (lane & 3),
                    be[r] * (xv[0][j][2 * r] - ee[r] * ak[0][j][2 * r]),
                    be[r] * (xv[0][j][2 * r + 1] - ee[r] * ak[0][j][2 * r + 1]));
    __syncthreads();
    zero(ak);
    mm(ak, t_a, x_b, m0, n0, 0, m0 + 16);  // U
    __syncthreads();
    each_pair(ak, m0, n0, [&](int i, int n, float x, float y) { put<2, PLX>(sx + i * LDX + n, x, y); });
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) aq[0][j][r] *= ee[r >> 1];
    __syncthreads();
    mm(aq, RowA<LDT, PLT, 2>(s.p), x_b, m0, n0, 0, m0 + 16);
    store_rows(aq, a.scale, o + vo + v0, vstride, rows, a.V - v0, m0, n0, width);
  }
}

template <class TI, int KP>
__global__ void __launch_bounds__(Out16<TI, KP>::NTH, Out16<TI, KP>::resident(sizeof(Out16<TI, KP>)))
    output16_kernel(Args a, const longlong2* __restrict__ tab, int VP, int tplanes, const bf* __restrict__ tinv,
                    const bf* __restrict__ states, TI* __restrict__ o) {
  griddep_launch_dependents();
  griddep_wait();
  output16_chunk<TI, KP>(a, tab, VP, tplanes, tinv, states, o);
  zero_uncovered(o, a, (int64_t)a.HV * a.V);
}

template <class TI, int KP, int NI>
int prep(const Args& a, const Saved& sv, int VP, float* b, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(Prep16<TI, KP, NI>);
  allow_smem<prep16_kernel<TI, KP, NI>>((int)smem);
  launch_pdl(prep16_kernel<TI, KP, NI>, dim3((unsigned)items), dim3(THREADS), smem, st, a, sv.chunk_tab, VP, (bf*)sv.tinv, sv.pm, b);
  SSLA_CHECK_LAUNCH("gated_delta_rule prep");
  return SSLA_OK;
}

template <class TI, int KP>
int output(const Args& a, const Saved& sv, int VP, bool exact, void* o, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(Out16<TI, KP>);
  allow_smem<output16_kernel<TI, KP>>((int)smem);
  launch_pdl(output16_kernel<TI, KP>, dim3((unsigned)items), dim3(Out16<TI, KP>::NTH), smem, st, a, sv.chunk_tab, VP, t_planes(exact), (const bf*)sv.tinv, (const bf*)sv.s, (TI*)o);
  SSLA_CHECK_LAUNCH("gated_delta_rule output");
  return SSLA_OK;
}

}  // namespace

int prep16(int dtype, const Args& a, const Saved& sv, int KP, int VP, bool exact, float* b, int64_t items,
           cudaStream_t st) {
  if (dtype == SSLA_F16)
    return KP == 64 ? prep<__half, 64, 3>(a, sv, VP, b, items, st) : prep<__half, 128, 3>(a, sv, VP, b, items, st);
  if (exact) return KP == 64 ? prep<bf, 64, 3>(a, sv, VP, b, items, st) : prep<bf, 128, 3>(a, sv, VP, b, items, st);
  return KP == 64 ? prep<bf, 64, 2>(a, sv, VP, b, items, st) : prep<bf, 128, 2>(a, sv, VP, b, items, st);
}

int output16(int dtype, const Args& a, const Saved& sv, int KP, int VP, bool exact, void* o, int64_t items,
             cudaStream_t st) {
  if (dtype == SSLA_F16)
    return KP == 64 ? output<__half, 64>(a, sv, VP, exact, o, items, st) : output<__half, 128>(a, sv, VP, exact, o, items, st);
  return KP == 64 ? output<bf, 64>(a, sv, VP, exact, o, items, st) : output<bf, 128>(a, sv, VP, exact, o, items, st);
}

}  // namespace delta
}  // namespace ssla
