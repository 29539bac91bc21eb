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

#include <type_traits>

#include "gemm_common.cuh"

namespace b200q {

constexpr int kMxTileRows = 128, kMxTileK = 256;
constexpr int kMxQBytes = 16384, kMxSfBytes = 1024, kMxTileBytes = kMxQBytes + kMxSfBytes;
constexpr int kMxBlockBytes = 17;  // ggml block_mxfp4: u8 e, u8 qs[16] (low nibbles elements 0..15, high nibbles 16..31)
constexpr int kMaxExperts = 1024, kMaxExpertsPerToken = 32;

inline __host__ __device__ int mx_k_tiles(int K) { return K / kMxTileK + (K % kMxTileK != 0); }
inline __host__ __device__ int64_t mx_row_tiles(int64_t rows) { return (rows + kMxTileRows - 1) / kMxTileRows; }
inline __host__ __device__ size_t mx_image_bytes(int64_t rows, int K) { return (size_t)mx_row_tiles(rows) * mx_k_tiles(K) * kMxTileBytes; }

// The grouping of token-expert pairs by expert (b200q_moe_plan), one buffer of int32. Pair s = t * k + j. A group's pairs keep
// their order; it is cut into tiles of 128, the row tiles of the activation image.
//   offsets[E + 1] | order[pairs] (pairs by expert, -1 behind the last) | place[pairs] (tile * 128 + row of pair s, or -1) |
//   n_tiles, n_units, 2 unused | tiles[max_tiles] {expert, first place in `order`, pairs, first pair}, 16-byte aligned |
//   units[max_units], two neighbouring tiles of an expert or its last one: {expert, first place, pairs, tile}, {first unit of the expert, its
//   units, 0, 0} | counts of the ranges
struct MoePlanLayout {
    size_t order, place, n_tiles, tiles, units, hist, total;
    int64_t max_tiles, max_units;
};
constexpr int kPlanRanges = 128;  // ranges of tokens that the grouping counts apart
inline __host__ MoePlanLayout moe_plan_layout(int64_t pairs, int E) {
    MoePlanLayout l;
    const int64_t met = pairs < E ? pairs : E;
    l.max_tiles = pairs / kMxTileRows + met;  // a group of c > 0 pairs has at most c / 128 + 1 tiles
    if (l.max_tiles > pairs) l.max_tiles = pairs;
    l.max_units = pairs / (2 * kMxTileRows) + met;
    if (l.max_units > pairs) l.max_units = pairs;
    l.order = (size_t)E + 1;
    l.place = l.order + (size_t)pairs;
    l.n_tiles = (l.place + (size_t)pairs + 3) & ~(size_t)3;
    l.tiles = l.n_tiles + 4;
    l.units = l.tiles + 4 * (size_t)l.max_tiles;
    l.hist = l.units + 8 * (size_t)l.max_units;
    l.total = l.hist + (size_t)kPlanRanges * (size_t)E;
    return l;
}

// Shared memory that a kernel with `cols` TMEM columns asks for, its own need being `bytes`: enough that the CTAs of clusters which an SM takes by its 228 KB always find their
// columns too, whichever of these kernels share it and whatever has come and gone. (A CTA that waits for columns while its cluster's others hold theirs could otherwise wait for
// a CTA that waits for it; one of no cluster comes to its end by itself.) 456 bytes a column, with the 2 KB of static and reserved memory, keep the sum at 512. Columns lie at
// multiples of their number, so that two CTAs of few could keep a third from its 256: 58 KB is more than half of what one of 256 leaves. (Without a cluster there may be more
// of them: 128256 x 512, one row, 10.7 us, with 58 KB each 12.9.)
inline size_t mx_smem_for_tmem(size_t bytes, uint32_t cols, bool cluster) {
    size_t least = (size_t)cols * 456 - 2048;
    if (cluster && least < 58 * 1024) least = 58 * 1024;
    return bytes < least ? least : bytes;
}

// A store of 32 bytes came with PTX ISA 8.8, that is CUDA 12.9. An older toolkit's ptxas refuses it; two of 16 bytes write the same.
#ifndef B200Q_STORE32
#if __CUDACC_VER_MAJOR__ > 12 || (__CUDACC_VER_MAJOR__ == 12 && __CUDACC_VER_MINOR__ >= 9)
#define B200Q_STORE32 1
#else
#define B200Q_STORE32 0
#endif
#endif

#ifdef __CUDACC__
// 32 bytes to a 32-byte aligned address
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&w)[8]) {
#if B200Q_STORE32
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
#else
    static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
#endif
}
__device__ __forceinline__ float e8m0_to_f32(uint32_t e) {  // 2^(e - 127); 0 is 2^-127, a subnormal
    return e == 255u ? __uint_as_float(0x7FC00000u) : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}
__device__ __forceinline__ size_t mx_tile_offset(int64_t row_tile, int k_tile, int k_tiles) { return ((size_t)row_tile * k_tiles + k_tile) * kMxTileBytes; }
__device__ __forceinline__ uint32_t mx_chunk_offset(int r, int b) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((b ^ (r & 7)) << 4)); }
__device__ __forceinline__ uint32_t mx_scale_offset(int r, int half) { return (uint32_t)(kMxQBytes + half * 512 + (r & 31) * 16 + (r >> 5) * 4); }
// Quantisation (OCP Microscaling Formats specification 1.0, 6.3): a block's exponent is floor(log2(largest magnitude)) - 2, which puts
// the largest magnitude into [4, 8); elements are divided by that power of two - exact in FP32 - and rounded to the nearest E2M1
// value, ties to the even one, magnitudes beyond 6 to 6. A block with an infinity or a NaN becomes NaN as a whole (e = 255), one of zeros e = 0.
// Eight neighbouring elements of a row as they lie in memory: four or eight registers.
template <typename T>
struct MxEight {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = ld_dep_u4(p + i * 16 / sizeof(T));
    }
    // Largest magnitude as the bits of an FP32: without their signs, bits compare like the magnitudes, infinities and NaNs above all. 16-bit types go two at a time.
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (sizeof(T) == 4) {
            const uint32_t m = 0x7FFFFFFFu;
            return max(max(max(q[0].x & m, q[0].y & m), max(q[0].z & m, q[0].w & m)), max(max(q[1].x & m, q[1].y & m), max(q[1].z & m, q[1].w & m)));
        } else {
            const uint32_t m = 0x7FFF7FFFu, two = __vmaxu2(__vmaxu2(q[0].x & m, q[0].y & m), __vmaxu2(q[0].z & m, q[0].w & m));
            const uint32_t one = max(two & 0xFFFFu, two >> 16);
            if constexpr (std::is_same_v<T, __nv_bfloat16>) return one << 16;
            else return __float_as_uint(h2f(one));
        }
    }
    __device__ __forceinline__ float get(int j) const {  // j is known when this is compiled
        const uint4& v = q[sizeof(T) == 4 ? j >> 2 : 0];
        const int i = sizeof(T) == 4 ? j & 3 : j >> 1;
        const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
        else return h2f(j & 1 ? w >> 16 : w & 0xFFFFu);
    }
};

// A quad of lanes holds a block, eight elements each: returns the lane's eight nibbles and the block's scale byte.
template <typename T>
__device__ __forceinline__ uint32_t mx_quantise8(const MxEight<T>& v, uint32_t& scale) {
    uint32_t top = v.top();
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
        : "f"(v.get(0) * inv), "f"(v.get(1) * inv), "f"(v.get(2) * inv), "f"(v.get(3) * inv), "f"(v.get(4) * inv), "f"(v.get(5) * inv), "f"(v.get(6) * inv), "f"(v.get(7) * inv));
    return out;
}

// Loads that do not go through the L1, for what is read ahead of griddepcontrol.wait.
__device__ __forceinline__ uint4 ld_l2_u4(const void* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_l2_u32(const void* p) {
    uint32_t v;
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

// ---- tcgen05 kind::mxf4 -----------------------------------------------------------------------------------------
// Operand without swizzle, rows of 16 bytes in groups of eight (128 bytes): the layout of a piece of scales.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}
// 32 rows x 16 bytes to four columns of TMEM, the same for each of the four lane quarters
template <int CG>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// kind::mxf4: A = B = E2M1 (1 at bits 7 and 10), scales E8M0 (bit 23), K-major, M = m, N = n, K = 64. `id` is the byte
// (0 or 2) of the 32-bit scale cells that holds the first of the two scales of a row.
__device__ __forceinline__ uint32_t instr_desc_mxf4(int m, int n, uint32_t id) {
    return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | (id << 29);
}
template <int CG>
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// ---- cluster ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mx_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mx_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t mx_map_to_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
// Arrives at another CTA's barrier, for what is asynchronous (kMbarOrder). (A release at this scope waits for all that the CTA has under way: by the relay of mx4_wide.cu,
// once a stage, it made 2000 x 14336 x 4096 90 us for 49, by its epilogue, once a tile, 53.)
__device__ __forceinline__ void mx_arrive_remote(uint32_t cluster_addr) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory"); }
// (relaxed: what the others have to see by then are barriers, which fence.mbarrier_init has released)
__device__ __forceinline__ void mx_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void mx_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(lds32(addr)); }
// A value to another CTA's shared memory; its barrier there counts the four bytes when they have arrived.
__device__ __forceinline__ void st_async_f32(uint32_t cluster_addr, float v, uint32_t cluster_bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(cluster_addr), "r"(__float_as_uint(v)), "r"(cluster_bar) : "memory");
}

// The roles that issue copies and MMAs run as whole warps with one elected lane at the instructions themselves: control flow, addresses and
// descriptors are then uniform for the compiler. (As code of one lane, every operand went through a conversion to a uniform register
// and a stage of the products took 1440 clocks to issue, 222 for a wait that had nothing to wait for.)
__device__ __forceinline__ int mx_uniform_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
__device__ __forceinline__ bool mx_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Bounded wait of a whole warp; false on all lanes once the CTA has given up.
template <MbarWait kWait = kMbarCta>
__device__ __forceinline__ bool mx_warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code, uint64_t limit_ns = kWaitLimitNs) {
    if (__all_sync(0xffffffffu, mbar_try_wait_as<kWait>(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait_or_abort_slow<kWait>(bar, parity, abort_flag, status, code, limit_ns) && !*abort_flag);
}

// silu(g) * u = g u / (1 + e^-g), from s = e^(-|g| / 2) <= 1: g / (1 + s s) or, for negative g, g s s / (1 + s s). Nothing leaves the range of the fast exponential and
// reciprocal. (From e^-g itself the quotient is 0 below g = -87.3, where e^-g passes 2^126; silu(-88) u need not be.) Off by |g| 2^-24 for the rounded argument, which only
// negative g feel, where silu is small, and 4.5 units of 2^-22: s by 1 twice, the reciprocal by a half, a sum and five products by a quarter each.
// (expf and a full division are 50 instructions a value: the gated tiles of mx4_wide.cu took 9000 clocks for the 8300 of their products.)
__device__ __forceinline__ float silu_times(float g, float u) {
    float s, inv;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(-0.721347520444481704f * fabsf(g)));  // log2(e) / 2
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(s, s, 1.f)));
    const float t = g < 0.f ? s : 1.f;
    return g * t * t * inv * u;
}
__device__ __forceinline__ float load_bias(const void* bias, int dtype, size_t i) {
    if (dtype == B200Q_DT_F32) return static_cast<const float*>(bias)[i];
    if (dtype == B200Q_DT_F16) return __half2float(static_cast<const __half*>(bias)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i]);
}
__device__ __forceinline__ void store_y(void* y, int dtype, size_t i, float v) {
    if (dtype == B200Q_DT_F32) static_cast<float*>(y)[i] = v;
    else if (dtype == B200Q_DT_F16) static_cast<__half*>(y)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}
#endif

}  // namespace b200q
