#pragma once
#include "delta_rule.cuh"

namespace ssla {
namespace delta {

// (I + A)^-1 of a 64 x 64 tile by one block of THREADS threads:
// sA strictly lower triangular -> sT, upper triangle zero; sY is scratch (>= 2048 floats).
// Diagonal 8 x 8 blocks by substitution (one thread a column, its block's entries in registers
// first), then pairs of blocks twice as large: the block below the diagonal is -T22 A21 T11.
__device__ __forceinline__ void unit_lower_inverse(const float* sA, float* sT, float* sY) {
  const int tid = threadIdx.x;
  for (int i = tid; i < BT * BT / 4; i += THREADS) {
    const int r = i >> 4, c = (i & 15) * 4;
    if ((r >> 3) != (c >> 3)) *reinterpret_cast<float4*>(sT + r * LDC + c) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (tid < 64) {
    const int b = tid & ~7, c = tid & 7;
    float a[8][8], x[8];
#pragma unroll
    for (int i = 1; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const float4 z = *reinterpret_cast<const float4*>(sA + (b + i) * LDC + b + j);
        a[i][j] = z.x; a[i][j + 1] = z.y; a[i][j + 2] = z.z; a[i][j + 3] = z.w;
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) x[i] = fmaf(-a[i][j], x[j], x[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sT[(b + i) * LDC + b + c] = x[i];
  }
  __syncthreads();
  {  // 8 -> 16, four pairs, 64 threads each: thread = (row, column)
    const int d = (tid >> 6) * 16, r = (tid >> 3) & 7, c = tid & 7;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x = fmaf(sA[(d + 8 + r) * LDC + d + j], sT[(d + j) * LDC + d + c], x);
    sY[tid] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) x = fmaf(-sT[(d + 8 + r) * LDC + d + 8 + j], sY[(tid & ~63) + j * 8 + c], x);
    __syncthreads();
    sT[(d + 8 + r) * LDC + d + c] = x;
  }
  __syncthreads();
  {  // 16 -> 32, two pairs, 128 threads each: thread = (row, 2 columns)
    const int p = tid >> 7, u = tid & 127, r = u >> 3, c = (u & 7) * 2, d = 32 * p;
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = sA[(d + 16 + r) * LDC + d + j];
      x = fmaf(a, sT[(d + j) * LDC + d + c], x);
      y = fmaf(a, sT[(d + j) * LDC + d + c + 1], y);
    }
    sY[p * 256 + r * 16 + c] = x;
    sY[p * 256 + r * 16 + c + 1] = y;
    __syncthreads();
    x = y = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = -sT[(d + 16 + r) * LDC + d + 16 + j];
      x = fmaf(a, sY[p * 256 + j * 16 + c], x);
      y = fmaf(a, sY[p * 256 + j * 16 + c + 1], y);
    }
    sT[(d + 16 + r) * LDC + d + c] = x;
    sT[(d + 16 + r) * LDC + d + c + 1] = y;
  }
  __syncthreads();
  {  // 32 -> 64: thread = 2 rows x 2 columns
    const int r = (tid >> 4) * 2, c = (tid & 15) * 2;
    float x[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const float a0 = sA[(32 + r) * LDC + j], a1 = sA[(33 + r) * LDC + j];
      const float b0 = sT[j * LDC + c], b1 = sT[j * LDC + c + 1];
      x[0][0] = fmaf(a0, b0, x[0][0]);
      x[0][1] = fmaf(a0, b1, x[0][1]);
      x[1][0] = fmaf(a1, b0, x[1][0]);
      x[1][1] = fmaf(a1, b1, x[1][1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sY[(r + i) * 33 + c + j] = x[i][j];
        x[i][j] = 0.f;
      }
    __syncthreads();
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const float a0 = -sT[(32 + r) * LDC + 32 + j], a1 = -sT[(33 + r) * LDC + 32 + j];
      const float b0 = sY[j * 33 + c], b1 = sY[j * 33 + c + 1];
      x[0][0] = fmaf(a0, b0, x[0][0]);
      x[0][1] = fmaf(a0, b1, x[0][1]);
      x[1][0] = fmaf(a1, b0, x[1][0]);
      x[1][1] = fmaf(a1, b1, x[1][1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) sT[(32 + r + i) * LDC + c + j] = x[i][j];
  }
  __syncthreads();
}

}  // namespace delta
}  // namespace ssla
