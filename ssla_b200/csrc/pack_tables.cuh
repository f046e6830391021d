// Chunk lists of packed sequences (cu_seqlens), built on the device so that no call reads back.
#pragma once
#include "common.cuh"

namespace ssla {
// Sequences are cut into chunks of `rows` tokens: chunk_off[n] (n <= N) is the first chunk of
// sequence n, chunk_tab[c] = {first token, tokens | sequence << 32} or {0, -1} behind the last one;
// MC >= (T + (rows - 1) N) / rows entries.  Offsets are clamped into [0, T] and the lists into their
// bounds, so malformed cu_seqlens cannot lead outside the buffers.
int launch_pack_tables(const int64_t* cu, int64_t N, int64_t T, int rows, int64_t MC, int* chunk_off,
                       longlong2* chunk_tab, cudaStream_t st);
}  // namespace ssla
