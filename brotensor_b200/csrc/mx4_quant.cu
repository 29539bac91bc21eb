// MXFP4 images: made from dense rows (quantise) or from a file's blocks (pack), and read back (dequantise).
// Bound by memory: 2 or 4 bytes in, 17/32 of a byte out per element, nothing is read twice.
#include "mx4_common.cuh"

namespace b200q {

constexpr int kQuantThreads = 256;

// Blocks of the three kernels cover a patch of rows x column tiles: of a block's eight warps 2^wide stand side by side along a row, the others
// on the rows below, and each takes `kBatch` neighbouring column tiles, whose loads are in flight together. No index needs a division (with
// one number per 256 columns, divided into row and column, the kernels ran at a quarter of the memory's rate).
struct Patch {
    int64_t row;
    int kt;
    __device__ __forceinline__ Patch(int wide, int batch) {
        const int warp = threadIdx.x >> 5;
        row = ((int64_t)blockIdx.x << (3 - wide)) + (warp >> wide);
        kt = (((int)blockIdx.y << wide) + (warp & ((1 << wide) - 1))) * batch;
    }
};

// A warp quantises 256 columns of a row: lane 4 b + s elements 8 s .. 8 s + 7 of block b. The row's 128 bytes of the image are
// one line. With `place`, row i of x is written to the rows place[i * copies + c], c < copies, of the image (-1: not).
// Dependents are let go once the predecessor has finished: what they read beside this kernel's results is then in place.
template <typename T, int kBatch>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantise_kernel(const T* x, int64_t rows, int K, int k_tiles, int wide, uint8_t* image, const int* place, int copies) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const Patch at(wide, kBatch);
    if (at.row >= rows || at.kt >= k_tiles) return;
    const T* src = x + at.row * K + (int64_t)at.kt * kMxTileK + 8 * lane;
    MxEight<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        v[u].clear();
        if ((at.kt + u) * kMxTileK + 8 * lane < K) v[u].load(src + u * kMxTileK);
    }
    uint32_t q[kBatch], word[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        uint32_t sc;
        q[u] = mx_quantise8(v[u], sc);
        // the four scales of the lane's half (blocks 0..3 or 4..7) in one word
        word[u] = sc << (8 * (b & 3));
        word[u] |= __shfl_xor_sync(0xffffffffu, word[u], 4);
        word[u] |= __shfl_xor_sync(0xffffffffu, word[u], 8);
    }
    for (int c = 0; c < copies; ++c) {
        const int64_t to = place ? (int64_t)(int)ld_dep_u32(place + at.row * copies + c) : at.row;
        if (to < 0) continue;
        const int r = (int)(to & 127);
        uint8_t* tile = image + mx_tile_offset(to >> 7, at.kt, k_tiles);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (at.kt + u < k_tiles) {
                *reinterpret_cast<uint32_t*>(tile + u * kMxTileBytes + mx_chunk_offset(r, b) + 4 * s) = q[u];
                if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + u * kMxTileBytes + mx_scale_offset(r, lane >> 4)) = word[u];
            }
        }
    }
}

template <typename T, int kBatch>
__global__ void __launch_bounds__(kQuantThreads) mx4_dequantise_kernel(const uint8_t* image, int64_t rows, int K, int k_tiles, int wide, T* out) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const Patch at(wide, kBatch);
    if (at.row >= rows || at.kt >= k_tiles) return;
    const int r = (int)(at.row & 127);
    const uint8_t* tile = image + mx_tile_offset(at.row >> 7, at.kt, k_tiles);
    uint32_t q[kBatch], word[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        q[u] = word[u] = 0u;
        if (at.kt + u < k_tiles) {
            q[u] = ld_dep_u32(tile + u * kMxTileBytes + mx_chunk_offset(r, b) + 4 * s);
            word[u] = ld_dep_u32(tile + u * kMxTileBytes + mx_scale_offset(r, b >> 2));
        }
    }
    T* dst = out + at.row * K + (int64_t)at.kt * kMxTileK + 8 * lane;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        if ((at.kt + u) * kMxTileK + 8 * lane >= K) continue;
        const float d = e8m0_to_f32(word[u] >> (8 * (b & 3)) & 255u);
        union {
            T e[8];
            uint4 v[sizeof(T) / 2];
        } o;
        uint32_t h[4];  // pairs of values in FP16, which holds them exactly
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(q[u]));
#pragma unroll
        for (int j = 0; j < 8; ++j) o.e[j] = from_f32<T>(h2f(j & 1 ? h[j >> 1] >> 16 : h[j >> 1] & 0xFFFFu) * d);
        uint4* to = reinterpret_cast<uint4*>(dst + u * kMxTileK);
        if (sizeof(T) == 4 && (reinterpret_cast<uintptr_t>(out) & 31) == 0) {  // whole sectors; two 16-byte stores leave halves
            const uint4 lo = o.v[0], hi = o.v[sizeof(T) / 2 - 1];
            st_global_32(to, {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
        } else {
#pragma unroll
            for (int j = 0; j < (int)(sizeof(T) / 2); ++j) to[j] = o.v[j];
        }
    }
}

// A file's blocks -> image. A warp moves 256 columns of a row: lane 4 b + s makes elements 8 s .. 8 s + 7 of block b, which are
// low (s < 2) or high nibbles of eight neighbouring bytes. `rows` of each of `count` matrices, each with an image of its own.
__global__ void __launch_bounds__(kQuantThreads) mx4_pack_kernel(const uint8_t* blocks, int64_t rows, int64_t count, int K, int k_tiles, int wide, uint8_t* image) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, b = lane >> 2, s = lane & 3;
    const Patch at(wide, 1);
    if (at.row >= rows * count || at.kt >= k_tiles) return;
    const int64_t mat = at.row / rows, row = at.row - mat * rows;
    const int r = (int)(row & 127);
    uint32_t q = 0, sc = 0;
    if (at.kt * kMxTileK + 32 * b < K) {
        const uint8_t* blk = blocks + ((size_t)at.row * (K / 32) + (size_t)at.kt * 8 + b) * kMxBlockBytes;
        sc = blk[0];
#pragma unroll
        for (int j = 0; j < 8; ++j) q |= ((uint32_t)blk[1 + 8 * (s & 1) + j] >> (s & 2 ? 4 : 0) & 15u) << (4 * j);
    }
    uint32_t word = sc << (8 * (b & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    uint8_t* tile = image + (size_t)mat * mx_image_bytes(rows, K) + mx_tile_offset(row >> 7, at.kt, k_tiles);
    *reinterpret_cast<uint32_t*>(tile + mx_chunk_offset(r, b) + 4 * s) = q;
    if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, lane >> 4)) = word;
}

// Warps side by side (2^wide of a block's eight) until a block's rows are all there are; blocks along the rows, and along the columns.
struct PatchGrid {
    dim3 grid;
    int wide;
    bool ok;
    PatchGrid(int64_t rows, int k_tiles, int batch) {
        const int64_t along = (k_tiles + batch - 1) / batch;
        wide = 0;
        while (wide < 3 && (2 << wide) <= along && rows <= (int64_t)4 >> wide) ++wide;
        const int64_t x = (rows + (8 >> wide) - 1) >> (3 - wide), y = (along + (1 << wide) - 1) >> wide;
        ok = x <= 2147483647LL && y <= 65535;
        grid = dim3((unsigned)x, (unsigned)y);
    }
};

template <typename T, int kBatch>
static int quantise_typed(const void* x, int64_t rows, int K, void* image, const int* place, int copies, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const PatchGrid g(rows, kt, kBatch);
    if (!g.ok) return fail(B200Q_ERR_UNSUPPORTED, "mx4_quantize: %lld x %d is more than one launch takes", (long long)rows, K);
    B200Q_CUDA_TRY(launch_dep(pdl_option() >= 0, mx4_quantise_kernel<T, kBatch>, g.grid, dim3(kQuantThreads), 0, st, static_cast<const T*>(x), rows, K, kt, g.wide,
                              static_cast<uint8_t*>(image), place, copies));
    return B200Q_OK;
}
template <typename T, int kBatch>
static int dequantise_typed(const void* image, int64_t rows, int K, void* out, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const PatchGrid g(rows, kt, kBatch);
    if (!g.ok) return fail(B200Q_ERR_UNSUPPORTED, "mx4_dequantize: %lld x %d is more than one launch takes", (long long)rows, K);
    B200Q_CUDA_TRY(launch_dep(pdl_option() >= 0, mx4_dequantise_kernel<T, kBatch>, g.grid, dim3(kQuantThreads), 0, st, static_cast<const uint8_t*>(image), rows, K, kt, g.wide,
                              static_cast<T*>(out)));
    return B200Q_OK;
}

// Several column tiles a warp once every SM has 32 warps' worth of single ones: four of 16-bit elements, two of FP32. Measured with two / four / eight (us):
// 14336 x 4096 BF16 30.7 / 25.5 / 24.6 and back 26.8 / 25.4 / 26.9, 2000 x 4096 BF16 5.4 / 5.2 / 6.2 and back 4.2 / 4.2 / 5.1, 2000 x 4096 FP32 6.5 / 6.8 / 7.7
// and back 6.0 / - / 8.2. 5.8 TB/s of read and written bytes on the first, where the loads' latency is what is left.
template <typename T>
constexpr int kBatchOf = sizeof(T) == 4 ? 2 : 4;

int launch_mx4_quantise(const void* x, int x_dtype, int64_t rows, int K, void* image, const int* place, int copies, int sms, cudaStream_t st) {
    const bool many = rows * mx_k_tiles(K) > (int64_t)sms * 32;
    auto run = [&](auto zero) {
        using T = decltype(zero);
        return many ? quantise_typed<T, kBatchOf<T>>(x, rows, K, image, place, copies, st) : quantise_typed<T, 1>(x, rows, K, image, place, copies, st);
    };
    return x_dtype == B200Q_DT_F32 ? run(0.f) : x_dtype == B200Q_DT_F16 ? run(__half()) : run(__nv_bfloat16());
}

int launch_mx4_dequantise(const void* image, int64_t rows, int K, void* out, int out_dtype, int sms, cudaStream_t st) {
    const bool many = rows * mx_k_tiles(K) > (int64_t)sms * 32;
    auto run = [&](auto zero) {
        using T = decltype(zero);
        return many ? dequantise_typed<T, kBatchOf<T>>(image, rows, K, out, st) : dequantise_typed<T, 1>(image, rows, K, out, st);
    };
    return out_dtype == B200Q_DT_F32 ? run(0.f) : out_dtype == B200Q_DT_F16 ? run(__half()) : run(__nv_bfloat16());
}

int launch_mx4_pack(const void* blocks, int64_t rows, int64_t count, int K, void* image, cudaStream_t st) {
    const int kt = mx_k_tiles(K);
    const PatchGrid g(rows * count, kt, 1);
    if (!g.ok) return fail(B200Q_ERR_UNSUPPORTED, "mx4_pack: %lld x %lld x %d is more than one launch takes", (long long)count, (long long)rows, K);
    B200Q_CUDA_TRY(launch_dep(pdl_option() >= 0, mx4_pack_kernel, g.grid, dim3(kQuantThreads), 0, st, static_cast<const uint8_t*>(blocks), rows, count, K, kt, g.wide,
                              static_cast<uint8_t*>(image)));
    return B200Q_OK;
}

}  // namespace b200q
