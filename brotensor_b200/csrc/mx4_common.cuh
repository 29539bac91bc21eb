// MXFP4: 32 neighbouring elements of a row share the scale 2^(e - 127) (one byte, E8M0; 255 is NaN), an element is
// 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign (four bits, E2M1). Layout of such a matrix on the device, the "image", and what
// the kernels on it share.
//
// The image is a row of tiles of 128 matrix rows x 256 columns, 17408 bytes each, all column tiles of a row tile one
// after the other: 16384 bytes of elements as a K-major tcgen05 operand with the 128-byte swizzle (row r at
// (r / 8) * 1024 + (r % 8) * 128, its block of 32 elements number b as the 16-byte chunk b ^ (r % 8), the even element
// of a pair in the low nibble), then two 512-byte pieces of scales, one per 128 columns, as tcgen05.cp 32x128b takes them (row r's
// four bytes at (r % 32) * 16 + (r / 32) * 4). A pipeline stage is therefore one contiguous bulk copy whatever the
// matrix: no tensor map, every address a multiple of 1024, and a weight matrix streams from HBM in order.
// Columns beyond K in the last tile hold zeros; rows beyond the last are not specified (nothing of a row reaches
// another row's results).
#pragma once

#include "gemm_common.cuh"

namespace b200q {

constexpr int kMxTileRows = 128, kMxTileK = 256;
constexpr int kMxQBytes = 16384, kMxSfBytes = 1024, kMxTileBytes = kMxQBytes + kMxSfBytes;
constexpr int kMxBlockBytes = 17;  // ggml block_mxfp4: u8 e, u8 qs[16] (low nibbles elements 0..15, high nibbles 16..31)
constexpr int kMaxExperts = 1024, kMaxExpertsPerToken = 32;

inline __host__ __device__ int mx_k_tiles(int K) { return (K + kMxTileK - 1) / kMxTileK; }
inline __host__ __device__ int64_t mx_row_tiles(int64_t rows) { return (rows + kMxTileRows - 1) / kMxTileRows; }
inline __host__ __device__ size_t mx_image_bytes(int64_t rows, int K) { return (size_t)mx_row_tiles(rows) * mx_k_tiles(K) * kMxTileBytes; }

// The grouping of token-expert pairs by expert (b200q_moe_plan), one buffer of int32. Pair s = t * k + j. A group's pairs keep
// their order; it is cut into tiles of 128, the row tiles of the activation image.
//   offsets[E + 1] | order[pairs] (pairs by expert, -1 behind the last) | place[pairs] (tile * 128 + row of pair s, or -1) |
//   n_tiles, 3 unused | tiles[max_tiles] {expert, first place in `order`, pairs, 0}, 16-byte aligned | counts of the blocks
struct MoePlanLayout {
    size_t order, place, n_tiles, tiles, hist, total;
    int64_t max_tiles;
    int hist_blocks;
};
constexpr int kPlanBlockPairs = 1024;
inline __host__ MoePlanLayout moe_plan_layout(int64_t pairs, int E) {
    MoePlanLayout l;
    const int64_t met = pairs < E ? pairs : E;
    l.max_tiles = pairs / kMxTileRows + met;  // a group of c > 0 pairs has at most c / 128 + 1 tiles
    if (l.max_tiles > pairs) l.max_tiles = pairs;
    l.hist_blocks = (int)((pairs + kPlanBlockPairs - 1) / kPlanBlockPairs);
    l.order = (size_t)E + 1;
    l.place = l.order + (size_t)pairs;
    l.n_tiles = (l.place + (size_t)pairs + 3) & ~(size_t)3;
    l.tiles = l.n_tiles + 4;
    l.hist = l.tiles + 4 * (size_t)l.max_tiles;
    l.total = l.hist + (size_t)l.hist_blocks * (size_t)E;
    return l;
}

#ifdef __CUDACC__
__device__ __forceinline__ float e8m0_to_f32(uint32_t e) {  // 2^(e - 127); 0 is 2^-127, a subnormal
    return e == 255u ? __uint_as_float(0x7FC00000u) : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}
__device__ __forceinline__ float e2m1_to_f32(uint32_t nib) {
    const uint32_t m = nib & 7u;
    const float a = m < 2u ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
    return nib & 8u ? -a : a;
}
__device__ __forceinline__ size_t mx_tile_offset(int64_t row_tile, int k_tile, int k_tiles) { return ((size_t)row_tile * k_tiles + k_tile) * kMxTileBytes; }
__device__ __forceinline__ uint32_t mx_chunk_offset(int r, int b) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((b ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t mx_scale_offset(int r, int half) { return (uint32_t)(kMxQBytes + half * 512 + (r & 31) * 16 + (r >> 5) * 4); }
#endif

}  // namespace b200q
