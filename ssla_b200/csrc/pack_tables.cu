// Chunk lists of packed sequences: one block scans the chunk counts of 1024 sequences at a time,
// then every thread finds the owners of its list entries by bisection.
#include "pack_tables.cuh"

namespace ssla {
namespace {

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : (x > hi ? hi : x); }

__global__ void __launch_bounds__(1024) tables_kernel(const int64_t* __restrict__ cu, int64_t N, int64_t T, int R,
                                                      int64_t MC, int* chunk_off, longlong2* chunk_tab) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int KEPT = 1024;  // bounds of this many sequences stay in shared memory
  __shared__ int part[32], run, kept_off[KEPT + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) run = 0;
  __syncthreads();
  for (int64_t n0 = 0; n0 < N; n0 += 1024) {
    const int64_t n = n0 + tid;
    int c = 0;
    if (n < N) {
      const int64_t b = clamp64(cu[n], 0, T), e = clamp64(cu[n + 1], b, T);
      c = (int)((e - b + R - 1) / R);
    }
    int sum = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += x;
    }
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int a = part[lane];
      const int a0 = a;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, a, d);
        if (lane >= d) a += x;
      }
      part[lane] = a - a0;
    }
    __syncthreads();
    const int end = run + part[warp] + sum;
    // MC bounds well-formed sequences; the clamp keeps malformed offsets inside the buffers
    if (n < N) chunk_off[n] = (int)clamp64(end - c, 0, MC);
    __syncthreads();
    if (tid == 1023) run = end;
    __syncthreads();
  }
  if (tid == 0) chunk_off[N] = (int)clamp64(run, 0, MC);
  __threadfence_block();
  __syncthreads();
  const bool kept = N <= KEPT;
  if (kept) {
    for (int64_t n = tid; n <= N; n += 1024) kept_off[n] = chunk_off[n];
    __syncthreads();
  }
  const int* off = kept ? kept_off : chunk_off;
  const int total = off[N];
  for (int64_t c = tid; c < MC; c += 1024) {
    longlong2 e = make_longlong2(0, -1);
    if (c < total) {
      int64_t lo = 0, hi = N;  // last n with off[n] <= c
      while (hi - lo > 1) {
        const int64_t m = (lo + hi) >> 1;
        if (off[m] <= c) lo = m; else hi = m;
      }
      const int64_t b = clamp64(cu[lo], 0, T), t1 = clamp64(cu[lo + 1], b, T), t0 = b + (c - off[lo]) * R;
      const int64_t rows = t1 - t0 < R ? t1 - t0 : R;
      if (rows > 0) e = make_longlong2(t0, rows | (lo << 32));
    }
    chunk_tab[c] = e;
  }
}

}  // namespace

int launch_pack_tables(const int64_t* cu, int64_t N, int64_t T, int rows, int64_t MC, int* chunk_off,
                       longlong2* chunk_tab, cudaStream_t st) {
  launch_pdl(tables_kernel, dim3(1), dim3(1024), 0, st, cu, N, T, rows, MC, chunk_off, chunk_tab);
  SSLA_CHECK_LAUNCH("chunk tables");
  return SSLA_OK;
}

}  // namespace ssla
