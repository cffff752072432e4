// Packed layout of 4-bit weights [N, K], K a multiple of 128.
//
// A tile is 16 rows; a chunk is 512 elements of K (four K-blocks of 128), the
// last one of a row padded.  A tile's chunk is contiguous, 4352 bytes:
//   4 K-blocks x 64 lanes x 16 bytes of codes, then 64 lanes x 4 bytes of scales.
// Lane l of a K-block holds row l % 16, elements 32 * (l / 16) .. +32 (two a
// byte, the lower index in the low half): the A operand of
// v_mfma_scale_f32_16x16x128_f8f6f4 with fp4 elements.  Byte b of a lane's
// scales is the e8m0 scale of those 32 elements in K-block b, which the
// instruction picks by its scale-select field: one dword load serves four.
// A tile's chunks follow each other, then the next tile's, so that a wave
// streams one contiguous run.
//
// The B operand (e4m3) of the same instruction: lane l holds column l % 16, in
// its first 16 bytes elements 16 * (l / 16) .. +16 and in its second
// 64 + 16 * (l / 16) .. +16.
#pragma once

#include "common.h"

#ifdef __HIPCC__
#define W4_HD __host__ __device__ __forceinline__
#else
#define W4_HD inline
#endif

namespace moe {

constexpr int W4_CHUNK_BLOCKS = 4;
constexpr int W4_CHUNK_K = W4_CHUNK_BLOCKS * BLK;
constexpr int W4_BLOCK_BYTES = 16 * BLK / 2;  // 1 KB
constexpr int W4_CHUNK_BYTES = W4_CHUNK_BLOCKS * W4_BLOCK_BYTES + 64 * 4;

W4_HD int w4_tiles(int N) { return (N + 15) / 16; }
W4_HD int w4_chunks(int K) { return (K + W4_CHUNK_K - 1) / W4_CHUNK_K; }

}  // namespace moe
