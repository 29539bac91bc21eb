// MXFP4 images: made from dense rows (quantise) or from a file's blocks (pack), and read back (dequantise).
//
// Quantisation (OCP Microscaling Formats specification 1.0, 6.3): a block's exponent is floor(log2(largest magnitude)) - 2, which puts
// the largest magnitude into [4, 8); elements are divided by that power of two - exact in FP32 - and rounded to the nearest E2M1
// value, ties to the even one, magnitudes beyond 6 to 6. A block with an infinity or a NaN becomes NaN as a whole (e = 255), one of zeros e = 0.
// Bound by memory: 2 or 4 bytes in, 17/32 of a byte out per element, nothing is read twice.
#include "mx4_common.cuh"

namespace b200q {

constexpr int kQuantThreads = 256;

// Eight neighbouring elements in FP32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = ld_dep_f4(p), b = ld_dep_f4(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        union {
            uint4 q;
            T e[8];
        } u;
        u.q = ld_dep_u4(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(u.e[i]);
    }
}

// A quad of lanes holds a block, eight elements each: returns the lane's eight nibbles and the block's scale byte.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], uint32_t& scale) {
    uint32_t top = 0;  // magnitudes as bits compare like magnitudes, infinities and NaNs above all
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int be = (int)(top >> 23);  // 0: a zero or a subnormal, below 2^-126 - the smallest scale serves
    if (be == 255) {
        scale = 255u;
        return 0u;
    }
    const int e = max(be - 2, 0);  // biased exponent of the scale
    scale = (uint32_t)e;
    // 1 / scale = 2^(127 - e), 127 - e in -125 .. 127
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    uint32_t out;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(out)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv), "f"(v[6] * inv), "f"(v[7] * inv));
    return out;
}

// A warp quantises 256 columns of a row: lane 4 b + s elements 8 s .. 8 s + 7 of block b. The row's 128 bytes of the image are
// one line. With `place`, row i of x is written to the rows place[i * copies + c], c < copies, of the image (-1: not).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantise_kernel(const T* x, int64_t rows, int K, int k_tiles, uint8_t* image, const int* place, int copies) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const int64_t items = rows * k_tiles, warps = (int64_t)gridDim.x * (kQuantThreads / 32);
    constexpr int kBatch = 4;  // items whose loads are in flight together
    for (int64_t i0 = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); i0 < items; i0 += warps * kBatch) {
        float v[kBatch][8];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t i = i0 + u * warps, row = i / k_tiles;
            const int k = (int)(i - row * k_tiles) * kMxTileK + 8 * lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
            if (i < items && k < K) load8(x + row * K + k, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t i = i0 + u * warps;
            if (i >= items) break;
            const int64_t row = i / k_tiles;
            const int kt = (int)(i - row * k_tiles);
            uint32_t sc;
            const uint32_t q = quantise8(v[u], sc);
            // the four scales of the lane's half (blocks 0..3 or 4..7) in one word
            uint32_t word = sc << (8 * (b & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            for (int c = 0; c < (place ? copies : 1); ++c) {
                const int64_t to = place ? (int64_t)(int)ld_dep_u32(place + row * copies + c) : row;
                if (to < 0) continue;
                uint8_t* tile = image + mx_tile_offset(to >> 7, kt, k_tiles);
                const int r = (int)(to & 127);
                *reinterpret_cast<uint32_t*>(tile + mx_chunk_offset(r, b) + 4 * s) = q;
                if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, lane >> 4)) = word;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) mx4_dequantise_kernel(const uint8_t* image, int64_t rows, int K, int k_tiles, T* out) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const int64_t items = rows * k_tiles, warps = (int64_t)gridDim.x * (kQuantThreads / 32);
    for (int64_t i = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); i < items; i += warps) {
        const int64_t row = i / k_tiles;
        const int kt = (int)(i - row * k_tiles), k = kt * kMxTileK + 8 * lane, r = (int)(row & 127);
        if (k >= K) continue;
        const uint8_t* tile = image + mx_tile_offset(row >> 7, kt, k_tiles);
        const uint32_t q = ld_dep_u32(tile + mx_chunk_offset(r, b) + 4 * s);
        const float d = e8m0_to_f32(ld_dep_u32(tile + mx_scale_offset(r, b >> 2)) >> (8 * (b & 3)) & 255u);
        union {
            T e[8];
            uint4 v[sizeof(T) / 2];
        } o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.e[j] = from_f32<T>(e2m1_to_f32(q >> (4 * j) & 15u) * d);
        uint4* dst = reinterpret_cast<uint4*>(out + row * K + k);
#pragma unroll
        for (int j = 0; j < (int)(sizeof(T) / 2); ++j) dst[j] = o.v[j];
    }
}

// A file's blocks -> image. A warp moves 256 columns of a row: lane 4 b + s makes elements 8 s .. 8 s + 7 of block b, which are
// low (s < 2) or high nibbles of eight neighbouring bytes. `rows` of each of `count` matrices, each with an image of its own.
__global__ void __launch_bounds__(kQuantThreads) mx4_pack_kernel(const uint8_t* blocks, int64_t rows, int64_t count, int K, int k_tiles, uint8_t* image) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const int64_t items = count * rows * k_tiles, warps = (int64_t)gridDim.x * (kQuantThreads / 32);
    const size_t bytes = mx_image_bytes(rows, K);
    for (int64_t i = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); i < items; i += warps) {
        const int64_t at = i / k_tiles, mat = at / rows, row = at - mat * rows;
        const int kt = (int)(i - at * k_tiles), r = (int)(row & 127);
        uint32_t q = 0, sc = 0;
        if (kt * kMxTileK + 32 * b < K) {
            const uint8_t* blk = blocks + ((size_t)at * (K / 32) + (size_t)kt * 8 + b) * kMxBlockBytes;
            sc = blk[0];
#pragma unroll
            for (int j = 0; j < 8; ++j) q |= ((uint32_t)blk[1 + 8 * (s & 1) + j] >> (s & 2 ? 4 : 0) & 15u) << (4 * j);
        }
        uint32_t word = sc << (8 * (b & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        uint8_t* tile = image + (size_t)mat * bytes + mx_tile_offset(row >> 7, kt, k_tiles);
        *reinterpret_cast<uint32_t*>(tile + mx_chunk_offset(r, b) + 4 * s) = q;
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, lane >> 4)) = word;
    }
}

static unsigned quant_grid(int64_t items, int batch, int sms) {
    const int64_t blocks = (items + (int64_t)batch * (kQuantThreads / 32) - 1) / (batch * (kQuantThreads / 32)), most = (int64_t)sms * 8;
    return (unsigned)(blocks < most ? blocks : most);
}

int launch_mx4_quantise(const void* x, int x_dtype, int64_t rows, int K, void* image, const int* place, int copies, int sms, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const int64_t items = rows * kt;
    // few items: one each per warp, so that they spread over the SMs
    const dim3 grid(quant_grid(items, items > (int64_t)sms * 32 ? 4 : 1, sms)), block(kQuantThreads);
    const bool dep = pdl_option() >= 0;
    uint8_t* im = static_cast<uint8_t*>(image);
    if (x_dtype == B200Q_DT_F32) B200Q_CUDA_TRY(launch_dep(dep, mx4_quantise_kernel<float>, grid, block, 0, st, static_cast<const float*>(x), rows, K, kt, im, place, copies));
    else if (x_dtype == B200Q_DT_F16) B200Q_CUDA_TRY(launch_dep(dep, mx4_quantise_kernel<__half>, grid, block, 0, st, static_cast<const __half*>(x), rows, K, kt, im, place, copies));
    else B200Q_CUDA_TRY(launch_dep(dep, mx4_quantise_kernel<__nv_bfloat16>, grid, block, 0, st, static_cast<const __nv_bfloat16*>(x), rows, K, kt, im, place, copies));
    return B200Q_OK;
}

int launch_mx4_dequantise(const void* image, int64_t rows, int K, void* out, int out_dtype, int sms, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const dim3 grid(quant_grid(rows * kt, 1, sms)), block(kQuantThreads);
    const bool dep = pdl_option() >= 0;
    const uint8_t* im = static_cast<const uint8_t*>(image);
    if (out_dtype == B200Q_DT_F32) B200Q_CUDA_TRY(launch_dep(dep, mx4_dequantise_kernel<float>, grid, block, 0, st, im, rows, K, kt, static_cast<float*>(out)));
    else if (out_dtype == B200Q_DT_F16) B200Q_CUDA_TRY(launch_dep(dep, mx4_dequantise_kernel<__half>, grid, block, 0, st, im, rows, K, kt, static_cast<__half*>(out)));
    else B200Q_CUDA_TRY(launch_dep(dep, mx4_dequantise_kernel<__nv_bfloat16>, grid, block, 0, st, im, rows, K, kt, static_cast<__nv_bfloat16*>(out)));
    return B200Q_OK;
}

int launch_mx4_pack(const void* blocks, int64_t rows, int64_t count, int K, void* image, int sms, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const dim3 grid(quant_grid(count * rows * kt, 1, sms)), block(kQuantThreads);
    B200Q_CUDA_TRY(launch_dep(pdl_option() >= 0, mx4_pack_kernel, grid, block, 0, st, static_cast<const uint8_t*>(blocks), rows, count, K, kt, static_cast<uint8_t*>(image)));
    return B200Q_OK;
}

}  // namespace b200q
