// Chunked gated delta rule, forward (delta_rule.cuh has the formulas).
//   tables      chunk and segment lists of the packed sequences (device only, no host read)
//   prep        per (chunk, value head): T, PM = Kl^T W, B = Kl^T T beta V, exp(gC)
//   chain       S' = exp(gC) S - PM S + B along every sequence: the one sequential part
//   output      per (chunk, value head): O from the start state
#include "delta_rule_16.cuh"
#include "delta_rule_inverse.cuh"
#include "pack_tables.cuh"

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
  Gates gates;
};

template <int KP>
__global__ void __launch_bounds__(THREADS, 2) prep_kernel(Args a, const longlong2* __restrict__ tab, int VP,
                                                          float* __restrict__ decay, float* __restrict__ tinv,
                                                          float* __restrict__ pm, float* __restrict__ bout) {
  using S = PrepSmem<KP>;
  constexpr bool X = false, SP = true;
  constexpr int LDK = S::LDK, LDV = S::LDV;
  extern __shared__ __align__(16) unsigned char raw[];
  S& s = *reinterpret_cast<S*>(raw);
  const int64_t chunk = blockIdx.x / a.HV;
  const int hv = (int)(blockIdx.x - chunk * a.HV), h = hv / a.R;
  const size_t item = blockIdx.x;
  int64_t t0;
  int rows;
  if (!locate(tab, a.MC, chunk, t0, rows)) return;
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
  if (threadIdx.x == 0) decay[item] = s.gates.whole;
  const TI* sk = s.k;
  const int m0 = (warp >> 1) * 16, n0 = (warp & 1) * 32;
  {
    float acc[1][4][4];
    zero(acc);
    if (n0 <= m0)
      warp_mma<X, X, SP>(acc, m0, n0, 0, KP, [&](int m, int k) { return pair(sk + m * LDK + k); },
                         [&](int k, int n) { return pair(sk + n * LDK + k); });
    each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
      const float b = s.gates.beta[i];
      s.a[i * LDC + j] = i > j ? b * s.gates.fade(i, j) * x : 0.f;
      s.a[i * LDC + j + 1] = i > j + 1 ? b * s.gates.fade(i, j + 1) * y : 0.f;
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
        warp_mma<false, X, SP>(acc, m0, n0, 0, m0 + 16, fa, [&](int j, int n) { return column<LDK>(sk + j * LDK + c0 + n); });
      else
        warp_mma<false, X, SP>(acc, m0, n0, 0, m0 + 16, fa, [&](int j, int n) { return column<LDV>(s.v + j * LDV + n); });
      each_pair(acc, m0, n0, [&](int i, int j, float x, float y) {
        const float l = s.gates.left[i];
        *reinterpret_cast<float2*>(s.y + i * 68 + j) = stage2<SP>(x * l, y * l);
      });
    }
    __syncthreads();
    {
      constexpr int MT = KP / 64;
      float acc[MT][4][4];
      zero(acc);
      const int mk = (warp >> 1) * 16 * MT;
      warp_mma<X, !SP, SP>(acc, mk, n0, 0, BT, [&](int m, int j) { return column<LDK>(sk + j * LDK + m); },
                           [&](int j, int n) { return column<68>(s.y + j * 68 + n); });
      float* out = w ? pm + item * KP * KP : bout + item * KP * VP;
      const int ld = w ? KP : VP;
      each_pair(acc, mk, n0, [&](int m, int n, float x, float y) {
        *reinterpret_cast<float2*>(out + (size_t)m * ld + c0 + n) = w ? stage2<SP>(x, y) : make_float2(x, y);
      });
    }
  }
}

// ------------------------------------------------------------------ chain
// One CTA carries VS columns of one state along its list of steps; every warp owns 16 of the KP
// rows in the accumulator layout.  A step needs one exchange of the state through shared memory
// (it is the right operand) and streams the step's [KP, KP] map through two cp.async buffers.
struct ChainArgs {
  const float* pm;        // [step * HV + hv][KP][KP]
  const float* b;         // [step * HV + hv][KP][VP]
  float* s;               // start state of every step ([..][KP][VP], two bf16 planes if planes); null: not kept
  const float* decay;     // per (step, hv); null: S' = PM S + B (composed maps)
  const int* off;         // steps of list n: off[n] .. off[n+1] - 1 ...
  const int4* seg;        // ... or of list n: seg[n].x, seg[n].y steps (seg[n].z < 0: none)
  const float* init;      // [n * HV + hv][K][V] unpadded (padded: [KP][VP])
  float* last;            // likewise
  float* mseg;            // composing: [n * HV + hv][KP][KP] for the columns from VP on, start from I
  bool init_padded, last_padded, reverse, compose, planes;
  int HV, K, V, VP, slices;
};

template <int KP, int VS, bool TRANS, bool SP>
__global__ void __launch_bounds__(KP * 2) chain_kernel(ChainArgs a) {
  constexpr int NTH = KP * 2, NT = VS / 8, LDP = KP + (TRANS ? 4 : 8), LDS = VS + 4;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sp = reinterpret_cast<float*>(raw);
  float* ss = sp + 2 * KP * LDP;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t lh = blockIdx.x / a.slices;
  int c0 = (int)(blockIdx.x - lh * a.slices) * VS;
  const int64_t list = lh / a.HV;
  const int hv = (int)(lh - list * a.HV);
  int first, count;
  if (a.seg) {
    const int4 e = a.seg[list];
    if (e.z < 0) return;
    first = e.x;
    count = e.y;
  } else {
    first = a.off[list];
    count = a.off[list + 1] - first;
  }
  const bool ident = a.compose && c0 >= a.VP;  // columns of the map itself
  if (ident) c0 -= a.VP;
  const int m0 = warp * 16;
  float S[1][NT][4];
  auto at = [&](int i) { return (int64_t)first + (a.reverse ? count - 1 - i : i); };
  auto load_map = [&](int i) {
    const float* src = a.pm + ((size_t)at(i) * a.HV + hv) * KP * KP;
    float* dst = sp + (i & 1) * KP * LDP;
    for (int j = threadIdx.x; j < KP * KP / 4; j += NTH) {
      const int r = j / (KP / 4), c = (j - r * (KP / 4)) * 4;
      cp16(dst + r * LDP + c, src + (size_t)r * KP + c);
    }
  };
  if (count > 0) load_map(0);
  cp_commit();
  // start state
  each_pair(S, m0, 0, [&](int r, int c, float& x, float& y) {
    x = y = 0.f;
    const int cc = c0 + c;
    if (ident) {
      x = r == cc ? 1.f : 0.f;
      y = r == cc + 1 ? 1.f : 0.f;
    } else if (a.init && a.init_padded) {
      const float2 z = *reinterpret_cast<const float2*>(a.init + ((size_t)lh * KP + r) * a.VP + cc);
      x = z.x;
      y = z.y;
    } else if (a.init && r < a.K) {
      const float* p = a.init + ((size_t)lh * a.K + r) * a.V + cc;
      if (cc < a.V) x = p[0];
      if (cc + 1 < a.V) y = p[1];
    }
  });
  float bn[NT][4];
  auto load_b = [&](int i) {
    const float* p = a.b + (((size_t)at(i) * a.HV + hv) * KP + m0) * a.VP + c0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float2 u = *reinterpret_cast<const float2*>(p + (size_t)g * a.VP + 8 * j + 2 * t);
      const float2 w = *reinterpret_cast<const float2*>(p + (size_t)(g + 8) * a.VP + 8 * j + 2 * t);
      bn[j][0] = u.x;
      bn[j][1] = u.y;
      bn[j][2] = w.x;
      bn[j][3] = w.y;
    }
  };
  float bc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) bc[j][0] = bc[j][1] = bc[j][2] = bc[j][3] = bn[j][0] = bn[j][1] = bn[j][2] = bn[j][3] = 0.f;
  if (!ident && count > 0) load_b(0);
  for (int i = 0; i < count; ++i) {
    const size_t it = (size_t)at(i) * a.HV + hv;
    float* sc = ss + (i & 1) * KP * LDS;
    each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
      *reinterpret_cast<float2*>(sc + r * LDS + c) = stage2<SP>(x, y);
    });
    const float d = a.decay ? a.decay[it] : 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) bc[j][r] = bn[j][r];
    if (a.s && !ident)
      each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
        if (a.planes)
          h16::put_at<2>((h16::bf*)a.s + (2 * it * KP + r) * a.VP + c0 + c, KP * a.VP, x, y);
        else
          *reinterpret_cast<float2*>(a.s + (it * KP + r) * a.VP + c0 + c) = make_float2(x, y);
      });
    cp_wait<0>();
    __syncthreads();  // map i and the state are there, step i - 1 is read
    if (i + 1 < count) {
      load_map(i + 1);
      if (!ident) load_b(i + 1);
    }
    cp_commit();
    const float* pc = sp + (i & 1) * KP * LDP;
    float acc[1][NT][4];
    zero(acc);
    warp_mma<!SP, !SP, SP>(acc, m0, 0, 0, KP,
                           [&](int m, int k) { return TRANS ? column<LDP>(pc + k * LDP + m) : pair(pc + m * LDP + k); },
                           [&](int k, int n) { return column<LDS>(sc + k * LDS + n); });
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S[0][j][r] = a.decay ? fmaf(d, S[0][j][r], bc[j][r] - acc[0][j][r]) : acc[0][j][r] + bc[j][r];
  }
  if (ident) {
    each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
      *reinterpret_cast<float2*>(a.mseg + ((size_t)lh * KP + r) * KP + c0 + c) = make_float2(x, y);
    });
  } else if (a.last && a.last_padded) {
    each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
      *reinterpret_cast<float2*>(a.last + ((size_t)lh * KP + r) * a.VP + c0 + c) = make_float2(x, y);
    });
  } else if (a.last) {
    each_pair(S, m0, 0, [&](int r, int c, float x, float y) {
      const int cc = c0 + c;
      if (r < a.K) {
        float* p = a.last + ((size_t)lh * a.K + r) * a.V + cc;
        if (cc < a.V) p[0] = x;
        if (cc + 1 < a.V) p[1] = y;
      }
    });
  }
}

template <int KP, int VS, bool TRANS, bool SP> int launch_chain(const ChainArgs& a, int64_t lists, cudaStream_t st) {
  constexpr size_t smem = 4 * (2 * KP * (KP + (TRANS ? 4 : 8)) + 2 * KP * (VS + 4));
  cudaFuncSetAttribute(chain_kernel<KP, VS, TRANS, SP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  const int64_t grid = lists * a.HV * a.slices;
  if (grid == 0) return SSLA_OK;
  chain_kernel<KP, VS, TRANS, SP><<<(unsigned)grid, KP * 2, smem, st>>>(a);
  SSLA_CHECK_LAUNCH("gated_delta_rule chain");
  return SSLA_OK;
}

template <int KP, int VS> int chain_vs(const ChainArgs& a, bool trans, bool split, int64_t lists, cudaStream_t st) {
  if (split) return trans ? launch_chain<KP, VS, true, true>(a, lists, st) : launch_chain<KP, VS, false, true>(a, lists, st);
  return trans ? launch_chain<KP, VS, true, false>(a, lists, st) : launch_chain<KP, VS, false, false>(a, lists, st);
}

template <int KP> int chain_kp(const ChainArgs& a, int vs, bool trans, bool split, int64_t lists, cudaStream_t st) {
  if (vs == 8) return chain_vs<KP, 8>(a, trans, split, lists, st);
  if (vs == 16) return chain_vs<KP, 16>(a, trans, split, lists, st);
  if (vs == 32) return chain_vs<KP, 32>(a, trans, split, lists, st);
  return chain_vs<KP, 64>(a, trans, split, lists, st);
}

int chain(ChainArgs a, int KP, int vs, bool trans, bool split, int64_t lists, cudaStream_t st) {
  a.slices = (a.VP + (a.compose ? KP : 0)) / vs;
  return KP == 64 ? chain_kp<64>(a, vs, trans, split, lists, st) : chain_kp<128>(a, vs, trans, split, lists, st);
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
  constexpr bool X = false, SP = true;
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
        warp_mma<X, X, SP>(acc, m0, p0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); },
                           [&](int k, int n) { return pair(sk + n * LDK + k); });
      each_pair(acc, m0, p0, [&](int i, int j, float x, float y) {
        *reinterpret_cast<float2*>(s.p + i * LDC + j) =
            stage2<SP>(i >= j ? s.gates.fade(i, j) * x : 0.f, i > j ? s.gates.fade(i, j + 1) * y : 0.f);
      });
    }
    cp_wait<0>();
    __syncthreads();
    float aq[1][NT][4], ak[1][NT][4];
    zero(aq);
    zero(ak);
    auto fs = [&](int k, int n) { return column<LDX>(s.s + k * LDX + n); };
    warp_mma<X, !SP, SP>(ak, m0, n0, 0, KP, [&](int m, int k) { return pair(sk + m * LDK + k); }, fs);
    warp_mma<X, !SP, SP>(aq, m0, n0, 0, KP, [&](int m, int k) { return pair(sq + m * LDK + k); }, fs);
    each_pair(ak, m0, n0, [&](int i, int n, float x, float y) {
      const float b = s.gates.beta[i], e = s.gates.start[i];
      *reinterpret_cast<float2*>(s.x + i * LDX + n) =
          stage2<SP>(b * (ldf(s.v + i * LDV + n) - e * x), b * (ldf(s.v + i * LDV + n + 1) - e * y));
    });
    __syncthreads();
    zero(ak);
    auto fx = [&](int k, int n) { return column<LDX>(s.x + k * LDX + n); };
    warp_mma<false, !SP, SP>(ak, m0, n0, 0, m0 + 16, [&](int m, int k) { return pair(s.t + m * LDC + k); }, fx);
    __syncthreads();
    each_pair(ak, m0, n0, [&](int i, int n, float x, float y) {
      *reinterpret_cast<float2*>(s.x + i * LDX + n) = stage2<SP>(x, y);
    });
    each_pair(aq, m0, n0, [&](int i, int, float& x, float& y) {
      x *= s.gates.start[i];
      y *= s.gates.start[i];
    });
    __syncthreads();
    warp_mma<!SP, !SP, SP>(aq, m0, n0, 0, m0 + 16, [&](int m, int k) { return pair(s.p + m * LDC + k); }, fx);
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
  output_chunk<KP, VB>(a, tab, VP, tinv, states, o);
  zero_uncovered(o, a, (int64_t)a.HV * a.V);
}

template <int KP>
int prep32(const Args& a, const Saved& sv, int VP, float* inc, int64_t items, cudaStream_t st) {
  const size_t smem = sizeof(PrepSmem<KP>);
  cudaFuncSetAttribute(prep_kernel<KP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  prep_kernel<KP><<<(unsigned)items, THREADS, smem, st>>>(a, sv.chunk_tab, VP, sv.decay, sv.tinv, sv.pm, inc);
  SSLA_CHECK_LAUNCH("gated_delta_rule prep");
  return SSLA_OK;
}

template <int KP>
int output32(const Args& a, const Saved& sv, int VP, void* o, int64_t items, cudaStream_t st) {
  constexpr int VB = KP == 64 ? 64 : 32;
  const size_t smem = sizeof(OutSmem<KP, VB>);
  cudaFuncSetAttribute(output_kernel<KP, VB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  output_kernel<KP, VB><<<(unsigned)items, THREADS, smem, st>>>(a, sv.chunk_tab, VP, sv.tinv, sv.s, (TI*)o);
  SSLA_CHECK_LAUNCH("gated_delta_rule output");
  return SSLA_OK;
}

}  // namespace

Plan make_plan(int64_t N, int64_t T, int64_t HV, int64_t K, int64_t V) {
  Plan p;
  p.MC = max_chunks(N, T);
  const int VP = pad_v(V), KP = pad_k(K);
  (void)KP;
  p.vs = 8;
  p.vs_seg = 16;
  while (p.vs < 64 && N * HV * (VP / p.vs) >= 4 * kNumSMs) p.vs *= 2;
  p.len = 0;
  p.MS = 0;
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
  SSLA_CHECK_ARG(N < (int64_t(1) << 31) && (max_chunks(N, T) + N) * (HV > 0 ? HV : 1) < (int64_t(1) << 26),
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
  c.HV = HV;
  c.K = K;
  c.V = V;
  c.VP = pad_v(V);
  c.reverse = reverse;
  c.planes = planes;
  const int KP = pad_k(K);
  c.pm = sv.pm;
  c.b = w.inc;
  c.s = s;
  c.decay = sv.decay;
  if (!p.len) {
    c.off = sv.chunk_off;
    c.init = init;
    c.last = last;
    return chain(c, KP, p.vs, reverse, exact, N, st);
  }
  // compose the maps of every segment, run along the segments, run inside them
  ChainArgs d = c;
  d.s = nullptr;
  d.seg = sv.seg_tab;
  d.compose = true;
  d.mseg = w.mseg;
  d.last = w.bseg;
  d.last_padded = true;
  int rc = chain(d, KP, p.vs_seg, reverse, exact, p.MS, st);
  if (rc) return rc;
  d = c;
  d.pm = w.mseg;
  d.b = d.s = w.bseg;
  d.decay = nullptr;
  d.off = sv.seg_off;
  d.init = init;
  d.last = last;
  d.planes = false;
  if ((rc = chain(d, KP, 16, false, exact, N, st))) return rc;
  c.seg = sv.seg_tab;
  c.init = w.bseg;
  c.init_padded = true;
  return chain(c, KP, p.vs_seg, reverse, exact, p.MS, st);
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
  SSLA_CHECK_ARG(T == 0 || (q && k && v && g && beta && o), "%s: null pointer", name);
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
  rc = launch_pack_tables(cu_seqlens, n_seqs, T, BT, p.MC, p.len, p.MS, sv.chunk_off, sv.seg_off, sv.chunk_tab,
                          sv.seg_tab, st);
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
  if (rc || T == 0) return rc;
  return !f32       ? output16(dtype, a, sv, KP, VP, exact, o, blocks, st)
         : KP == 64 ? output32<64>(a, sv, VP, o, blocks, st)
                    : output32<128>(a, sv, VP, o, blocks, st);
}
