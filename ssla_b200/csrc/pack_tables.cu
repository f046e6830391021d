// Chunk lists of packed sequences: one block scans the chunk counts of 1024 sequences at a time,
// then every thread finds the owners of its list entries by bisection.
#include "pack_tables.cuh"

namespace ssla {
namespace {

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : (x > hi ? hi : x); }

__global__ void __launch_bounds__(1024) tables_kernel(const int64_t* __restrict__ cu, int64_t N, int64_t T, int BT,
                                                      int64_t MC, int64_t len, int64_t MS, int* chunk_off, int* seg_off,
                                                      longlong2* chunk_tab, int4* seg_tab) {
  constexpr int KEPT = 1024;  // bounds of this many sequences stay in shared memory
  __shared__ int wc[32], ws[32], run[2], kc[KEPT + 1], ks[KEPT + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) run[0] = run[1] = 0;
  __syncthreads();
  for (int64_t n0 = 0; n0 < N; n0 += 1024) {
    const int64_t n = n0 + tid;
    int c = 0, g = 0;
    if (n < N) {
      const int64_t b = clamp64(cu[n], 0, T), e = clamp64(cu[n + 1], b, T);
      c = (int)((e - b + BT - 1) / BT);
      g = len ? (int)((c + len - 1) / len) : 0;
    }
    int sc = c, sg = g;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sc, d), y = __shfl_up_sync(0xffffffffu, sg, d);
      if (lane >= d) { sc += x; sg += y; }
    }
    if (lane == 31) { wc[warp] = sc; ws[warp] = sg; }
    __syncthreads();
    if (warp == 0) {
      int a = wc[lane], b = ws[lane];
      const int a0 = a, b0 = b;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, a, d), y = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= d) { a += x; b += y; }
      }
      wc[lane] = a - a0;
      ws[lane] = b - b0;
    }
    __syncthreads();
    const int ac = run[0] + wc[warp] + sc, ag = run[1] + ws[warp] + sg;
    if (n < N) {
      chunk_off[n] = (int)clamp64(ac - c, 0, MC);  // MC, MS bound well-formed sequences; the clamp keeps
      if (len) seg_off[n] = (int)clamp64(ag - g, 0, MS);    // malformed offsets inside the buffers
    }
    __syncthreads();
    if (tid == 1023) { run[0] = ac; run[1] = ag; }
    __syncthreads();
  }
  if (tid == 0) {
    chunk_off[N] = (int)clamp64(run[0], 0, MC);
    if (len) seg_off[N] = (int)clamp64(run[1], 0, MS);
  }
  __threadfence_block();
  __syncthreads();
  auto owner = [&](const int* off, int64_t c) {  // last n with off[n] <= c
    int64_t lo = 0, hi = N;
    while (hi - lo > 1) {
      const int64_t m = (lo + hi) >> 1;
      if (off[m] <= c) lo = m; else hi = m;
    }
    return lo;
  };
  const bool kept = N <= KEPT;
  if (kept) {
    for (int64_t n = tid; n <= N; n += 1024) {
      kc[n] = chunk_off[n];
      if (len) ks[n] = seg_off[n];
    }
    __syncthreads();
  }
  const int* oc = kept ? kc : chunk_off;
  const int* os = kept ? ks : seg_off;
  const int total = chunk_off[N], segs = len ? seg_off[N] : 0;
  for (int64_t c = tid; c < MC; c += 1024) {
    longlong2 e = make_longlong2(0, -1);
    if (c < total) {
      const int64_t n = owner(oc, c);
      const int64_t b = clamp64(cu[n], 0, T), t1 = clamp64(cu[n + 1], b, T), t0 = b + (c - oc[n]) * BT;
      const int64_t rows = t1 - t0 < BT ? t1 - t0 : BT;
      if (rows > 0) e = make_longlong2(t0, rows | (n << 32));
    }
    chunk_tab[c] = e;
  }
  for (int64_t s = tid; s < MS; s += 1024) {
    int4 e = make_int4(0, 0, -1, 0);
    if (s < segs) {
      const int n = (int)owner(os, s);
      const int first = oc[n] + (int)((s - os[n]) * len);
      int cnt = oc[n + 1] - first;
      cnt = cnt < 0 ? 0 : (cnt > len ? (int)len : cnt);
      e = make_int4(first, cnt, n, 0);
    }
    seg_tab[s] = e;
  }
}

}  // namespace

int launch_pack_tables(const int64_t* cu, int64_t N, int64_t T, int rows, int64_t MC, int64_t len, int64_t MS,
                       int* chunk_off, int* seg_off, longlong2* chunk_tab, int4* seg_tab, cudaStream_t st) {
  tables_kernel<<<1, 1024, 0, st>>>(cu, N, T, rows, MC, len, len ? MS : 0, chunk_off, seg_off, chunk_tab, seg_tab);
  SSLA_CHECK_LAUNCH("chunk tables");
  return SSLA_OK;
}

}  // namespace ssla
