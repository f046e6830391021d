// Products of the per-chunk kernels for 16-bit tokens (delta_rule_16.cu, delta_rule_16_bwd.cu).
//
// Every operand is a sum of bf16 planes: bf16 tokens are one plane, fp16 tokens two (exact),
// intermediate results x = p0 + p1 (+ p2), each plane the bf16 rounding of what the planes before
// leave, so two planes hold 16 bits and three 24.  A product keeps the plane pairs (i, j) with
// i + j < max(planes): 2 MMAs for token x 2 planes, 3 for 2 x 2, 3 for token x 3, 6 for 3 x 3.  The
// planes lie in shared memory as 16-bit tiles with rows 8 elements longer than the matrix (16-byte
// rows at odd multiples of 16: ldmatrix without bank conflicts), and ldmatrix with or without
// transposition reads either orientation of a tile as either operand, four 8x8 blocks an
// instruction.  Against TF32 products (11-bit operands of 4 bytes, one 32-bit load for every
// operand register) the same tensor time carries 16 bits with half the instructions; 8 x 2048
// tokens, 4 heads of 64: output went from 41 us on TF32 to 27 us, backward from 134 to 90 us.  What
// bounds them now is the dependent chain of a chunk's products (a barrier between each, two or three
// blocks an SM to hide it) and, at K = 128, shared-memory bandwidth next to the tensor pipe.
#pragma once
#include "delta_rule.cuh"

namespace ssla {
namespace delta {
namespace h16 {

using bf = __nv_bfloat16;
constexpr int LDT = BT + 8;  // rows of [64, 64] tiles

template <class TI> struct Planes;  // of a token tile
template <> struct Planes<__nv_bfloat16> { static constexpr int n = 1; };
template <> struct Planes<__half> { static constexpr int n = 2; };

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Left operand, 16 x 16 blocks at (m, k).  RowA: stored [m][k].  ColA: stored [k][m].
template <int LD, int PLANE, int N> struct RowA {
  static constexpr int n = N;
  uint32_t at;
  __device__ __forceinline__ RowA(const bf* p) {
    const int l = threadIdx.x & 31;
    at = smem_u32(p + (l & 15) * LD + (l >> 4) * 8);
  }
  __device__ __forceinline__ void load(uint32_t (&r)[4], int m, int k, int p) const {
    ldsm4(r, at + 2 * (p * PLANE + m * LD + k));
  }
};
template <int LD, int PLANE, int N> struct ColA {
  static constexpr int n = N;
  uint32_t at;
  __device__ __forceinline__ ColA(const bf* p) {
    const int l = threadIdx.x & 31;
    at = smem_u32(p + ((l & 7) + (l >> 4) * 8) * LD + ((l >> 3) & 1) * 8);
  }
  __device__ __forceinline__ void load(uint32_t (&r)[4], int m, int k, int p) const {
    ldsm4t(r, at + 2 * (p * PLANE + k * LD + m));
  }
};
// The 10 blocks of a lower triangular [64, 64] matrix as left operand fragments: [plane][block][lane]
// of 16 bytes, block (m, k) at m (m + 1) / 2 + k.  TR: the transpose, its 8 x 8 pieces turned in
// registers.
constexpr int FRAGS = 10 * 32, FRAG_BYTES = FRAGS * 16, FRAG_ELEMS = FRAG_BYTES / 2;  // of a plane
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int N, bool TR> struct FragA {
  static constexpr int n = N;
  const uint4* at;
  __device__ __forceinline__ FragA(const void* p) : at((const uint4*)p + (threadIdx.x & 31)) {}
  __device__ __forceinline__ void load(uint32_t (&r)[4], int m, int k, int p) const {
    const int i = (TR ? k : m) >> 4, j = (TR ? m : k) >> 4;
    const uint4 x = at[p * FRAGS + (i * (i + 1) / 2 + j) * 32];
    r[0] = TR ? turned(x.x) : x.x;
    r[1] = TR ? turned(x.z) : x.y;
    r[2] = TR ? turned(x.y) : x.z;
    r[3] = TR ? turned(x.w) : x.w;
  }
};
// Right operand, 16 x 16 blocks at (k, n).  RowB: stored [k][n].  ColB: stored [n][k].
template <int LD, int PLANE, int N> struct RowB {
  static constexpr int n = N;
  uint32_t at;
  __device__ __forceinline__ RowB(const bf* p) {
    const int l = threadIdx.x & 31;
    at = smem_u32(p + ((l & 7) + ((l >> 3) & 1) * 8) * LD + (l >> 4) * 8);
  }
  __device__ __forceinline__ void load(uint32_t (&r)[4], int k, int c, int p) const {
    ldsm4t(r, at + 2 * (p * PLANE + k * LD + c));
  }
};
template <int LD, int PLANE, int N> struct ColB {
  static constexpr int n = N;
  uint32_t at;
  __device__ __forceinline__ ColB(const bf* p) {
    const int l = threadIdx.x & 31;
    at = smem_u32(p + ((l & 7) + (l >> 4) * 8) * LD + ((l >> 3) & 1) * 8);
  }
  __device__ __forceinline__ void load(uint32_t (&r)[4], int k, int c, int p) const {
    ldsm4(r, at + 2 * (p * PLANE + c * LD + k));
  }
};

// The kept products of planes of one 16 x 16 block of A with two column tiles, small ones first.
template <int NA, int NB>
__device__ __forceinline__ void plane_products(float (&c0)[4], float (&c1)[4], const uint32_t (&fa)[NA][4],
                                               const uint32_t (&fb)[NB][4]) {
  constexpr int MOST = NA > NB ? NA : NB;
#pragma unroll
  for (int s = MOST - 1; s >= 0; --s)
#pragma unroll
    for (int p = 0; p <= s; ++p)
      if (p < NA && s - p < NB) {
        mma16(c0, fa[p], fb[s - p][0], fb[s - p][1]);
        mma16(c1, fa[p], fb[s - p][2], fb[s - p][3]);
      }
}
// all planes of a block of either operand
template <class A> __device__ __forceinline__ void planes_at(uint32_t (&f)[A::n][4], const A& a, int i, int j) {
#pragma unroll
  for (int p = 0; p < A::n; ++p) a.load(f[p], i, j, p);
}

// acc += A B over k in [k0, k1) (multiples of 16), columns n0 .. n0 + 8 NT
template <int MT, int NT, class A, class B>
__device__ __forceinline__ void mm(float (&acc)[MT][NT][4], const A& a, const B& b, int m0, int n0, int k0, int k1) {
  static_assert(NT % 2 == 0, "columns come in pairs of tiles");
#pragma unroll 4
  for (int k = k0; k < k1; k += 16) {
    uint32_t fa[MT][A::n][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) planes_at(fa[i], a, m0 + 16 * i, k);
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      uint32_t fb[B::n][4];
      planes_at(fb, b, k, n0 + 8 * j);
#pragma unroll
      for (int i = 0; i < MT; ++i) plane_products<A::n, B::n>(acc[i][j], acc[i][j + 1], fa[i], fb);
    }
  }
}
// Two left operands with one right operand, read once: the loads of shared memory are what these
// kernels wait for beside the tensor pipe.
template <int NT, class A, class C, class B>
__device__ __forceinline__ void mm_ab_cb(float (&x)[1][NT][4], const A& a, float (&y)[1][NT][4], const C& c, const B& b,
                                         int m0, int n0, int k0, int k1) {
#pragma unroll 4
  for (int k = k0; k < k1; k += 16) {
    uint32_t fa[A::n][4], fc[C::n][4];
    planes_at(fa, a, m0, k);
    planes_at(fc, c, m0, k);
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      uint32_t fb[B::n][4];
      planes_at(fb, b, k, n0 + 8 * j);
      plane_products<A::n, B::n>(x[0][j], x[0][j + 1], fa, fb);
      plane_products<C::n, B::n>(y[0][j], y[0][j + 1], fc, fb);
    }
  }
}
// One left operand with two right operands.
template <int NT, class A, class B, class C>
__device__ __forceinline__ void mm_ab_ac(float (&x)[1][NT][4], const B& b, float (&y)[1][NT][4], const C& c, const A& a,
                                         int m0, int n0, int k0, int k1) {
#pragma unroll 4
  for (int k = k0; k < k1; k += 16) {
    uint32_t fa[A::n][4];
    planes_at(fa, a, m0, k);
#pragma unroll
    for (int j = 0; j < NT; j += 2) {
      uint32_t fb[B::n][4], fc[C::n][4];
      planes_at(fb, b, k, n0 + 8 * j);
      planes_at(fc, c, k, n0 + 8 * j);
      plane_products<A::n, B::n>(x[0][j], x[0][j + 1], fa, fb);
      plane_products<A::n, C::n>(y[0][j], y[0][j + 1], fa, fc);
    }
  }
}

__device__ __forceinline__ uint32_t pack(float x, float y) {  // x in the low half
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void store2(__nv_bfloat16* p, float x, float y) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
}
__device__ __forceinline__ void store2(__half* p, float x, float y) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
}
// what the planes so far leave of x, y
__device__ __forceinline__ void rest(uint32_t w, float& x, float& y) {
  x -= __uint_as_float(w << 16);
  y -= __uint_as_float(w & 0xffff0000u);
}
// N planes of the pair (x, y) at p, plane elements apart
template <int N> __device__ __forceinline__ void put_at(bf* p, size_t plane, float x, float y) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t w = pack(x, y);
    *reinterpret_cast<uint32_t*>(p + i * plane) = w;
    if (i + 1 < N) rest(w, x, y);
  }
}
template <int N, int PLANE> __device__ __forceinline__ void put(bf* p, float x, float y) { put_at<N>(p, PLANE, x, y); }

// ------------------------------------------------------------------ token tiles
// dst[planes][64][LD] = rows of src (COLS columns, zeros behind); asynchronous for bf16.
template <class TI, int LD, int COLS, int NTH>
__device__ __forceinline__ void load_tokens(bf* dst, const TI* src, size_t stride, int rows, int cols, bool vec) {
  constexpr int PR = COLS / 8, PLANE = BT * LD;
  if constexpr (Planes<TI>::n == 1) {
    if (vec) {
      for (int i = threadIdx.x; i < BT * PR; i += NTH) {
        const int r = i / PR, c = (i % PR) * 8;
        if (r < rows && c < cols) cp16(dst + r * LD + c, src + r * stride + c);
        else *reinterpret_cast<uint4*>(dst + r * LD + c) = make_uint4(0, 0, 0, 0);
      }
      return;
    }
  }
  for (int i = threadIdx.x; i < BT * COLS / 2; i += NTH) {
    const int r = i / (COLS / 2), c = (i % (COLS / 2)) * 2;
    float x = 0.f, y = 0.f;
    if (r < rows) {
      const TI* p = src + r * stride + c;
      if (vec) {  // even columns, 4-byte aligned
        if (c < cols) {
          const float2 z = pair(p);
          x = z.x;
          y = z.y;
        }
      } else {
        if (c < cols) x = ldf(p);
        if (c + 1 < cols) y = ldf(p + 1);
      }
    }
    put<Planes<TI>::n, PLANE>(dst + r * LD + c, x, y);
  }
}
// planes of a state panel: dst[2][ROWS][LD], src [2][ROWS][stride] (16-byte aligned)
template <int LD, int ROWS, int COLS, int NTH>
__device__ __forceinline__ void load_planes(bf* dst, const bf* src, int stride) {
  constexpr int PR = COLS / 8;
  for (int i = threadIdx.x; i < 2 * ROWS * PR; i += NTH) {
    const int r = i / PR, c = (i % PR) * 8;
    cp16(dst + r * LD + c, src + (size_t)r * stride + c);
  }
}
template <int NTH> __device__ __forceinline__ void copy16(void* dst, const void* src, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += NTH * 16) cp16((char*)dst + i, (const char*)src + i);
}

__device__ __forceinline__ uint32_t pack_as(const __nv_bfloat16*, float x, float y) { return pack(x, y); }
__device__ __forceinline__ uint32_t pack_as(const __half*, float x, float y) {
  const __half2 v = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// How many elements of a result's rows (cols of them, stride a multiple of cols) one store can take.
__device__ __forceinline__ int store_width(const void* p, int cols) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  return cols % 8 == 0 && at % 16 == 0 ? 8 : cols % 2 == 0 && at % 4 == 0 ? 2 : 1;
}
// A warp's accumulator, times f, into rows [0, rows) and columns [0, cols) of a 16-bit result.  The two
// columns that a lane has of each 8-column tile are turned within quads into whole tiles: 16 bytes a
// store.  Piece q: row q / NT, tile q % NT.
template <class TO, int NT>
__device__ __forceinline__ void store_rows(const float (&acc)[1][NT][4], float f, TO* out, size_t stride, int rows,
                                           int cols, int m0, int n0, int width) {
  static_assert(NT % 2 == 0, "pieces come in fours");
  const int lane = threadIdx.x & 31, t = lane & 3, i0 = m0 + (lane >> 2);
  if (width == 8) {
#pragma unroll
    for (int u = 0; u < NT / 2; ++u) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = (4 * u + e) % NT, r = (4 * u + e) / NT;
        w[e] = pack_as(out, f * acc[0][j][2 * r], f * acc[0][j][2 * r + 1]);
      }
      quad_turn(w, t);
      const int q = 4 * u + t, i = i0 + 8 * (q / NT), c = n0 + 8 * (q % NT);
      if (i < rows && c < cols) *reinterpret_cast<uint4*>(out + i * stride + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = i0 + 8 * r, c = n0 + 8 * j + 2 * t;
      if (i >= rows || c >= cols) continue;
      TO* p = out + i * stride + c;
      const float x = f * acc[0][j][2 * r], y = f * acc[0][j][2 * r + 1];
      if (width == 2) {
        store2(p, x, y);
      } else {
        stf(p, x);
        if (c + 1 < cols) stf(p + 1, y);
      }
    }
}

// Pairs (row i, columns c, c + 1) of a token matrix in the accumulator layout, zeros outside: all
// loads before the first use.  even: an even number of columns, 4-byte aligned.
template <class TI, int NT>
__device__ __forceinline__ void load_pairs(float (&acc)[1][NT][4], const TI* src, size_t stride, int rows, int cols,
                                           int m0, int n0, bool even) {
  const int lane = threadIdx.x & 31, i0 = m0 + (lane >> 2), c0 = n0 + 2 * (lane & 3);
  uint32_t w[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = i0 + 8 * r, c = c0 + 8 * j;
      const TI* p = src + i * stride + c;
      w[j][r] = 0;
      if (even) {
        if (i < rows && c < cols) w[j][r] = __ldg(reinterpret_cast<const unsigned*>(p));
      } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        if (i < rows && c < cols) w[j][r] = __ldg(q);
        if (i < rows && c + 1 < cols) w[j][r] |= (uint32_t)__ldg(q + 1) << 16;
      }
    }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 z = pair(reinterpret_cast<const TI*>(&w[j][r]));
      acc[0][j][2 * r] = z.x;
      acc[0][j][2 * r + 1] = z.y;
    }
}

}  // namespace h16
}  // namespace delta
}  // namespace ssla
