// Products of MXFP4 images where there are many activation rows: the arithmetic of mx4_gemm.cu on tiles of 256 weight rows, activations
// as the MMA's M, so that a thread of the epilogue holds one result row and stores 32 bytes of it at a time (weight rows as M, as the
// small kernel has them, is 128 two-byte stores per thread and tile: 14 us of a 23 us tile at K = 4096).
//
// A pair of CTAs runs one tcgen05.mma.cta_group::2 of 256 activation rows x 256 weight rows; each CTA fetches its 128
// activation rows and half of the weight rows (the scales of all 256), 35 KB per 256 columns and SM. One CTA on 128 x 256 would fetch 51 KB for the
// same work per SM, and the operand stream from the L2 (about 12 TB/s) is what bounds these tiles.
// The two halves of the weight rows are two row tiles of one matrix, or (GATED) the same row tile of gate and up: columns c and
// 128 + c of the accumulator then meet in silu(gate) * up in the thread that holds both.
//
// Persistent CTAs; the ring runs on across tiles, so that the next tile's operands arrive while this one's results leave. 256 columns of TMEM are
// the accumulator and 24 per stage hold scales, which leaves no room for a second accumulator: the eight epilogue warps take the whole tile
// into registers first (128 values a thread), give the accumulator back and convert and store while the next tile runs.
//   warp 0  loader    warp 1  TMEM, MMAs (the pair's leader)    warp 2  relay: this CTA's stage has landed -> leader
//   warps 4..11  epilogue
#include "mx4_common.cuh"

namespace b200q {

constexpr int kWideThreads = 384, kWideEpilogueWarp0 = 4, kWideStages = 6;
// [activations and their scales][half of the weight rows][scales of all weight rows]
constexpr int kWideStageBytes = kMxTileBytes + kMxQBytes + 2 * kMxSfBytes;
constexpr int kWideSfCols = 24;  // per stage: 8 TMEM columns of activations' scales, 16 of weights'

struct WideParams {
    const uint8_t* W;      // image of the (gate) weights; expert e's lies e * w_expert_bytes behind
    const uint8_t* W_up;
    const uint8_t* X;
    const void* bias;
    void* Y;
    int* status;
    size_t w_expert_bytes;
    const int4* units;     // grouped: {expert, first place, rows, first tile}, {first unit, units of the expert, ..} of two neighbouring tiles; nullptr: one matrix
    const int* n_units;
    const int* order;
    int M, N, K, k_tiles;
    int row_tiles;         // 128-row tiles of a weight matrix
    int w_tiles;           // 256-wide tiles of results: pairs of row tiles, or (gated) row tiles
    int bias_dtype, y_dtype;
    int early;             // the predecessor writes neither weights nor plan (it is the quantisation): they are read ahead of its end
};

__device__ __forceinline__ void wide_alloc(uint32_t slot) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void wide_dealloc(uint32_t base) { asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory"); }
// arrives on the barrier in both CTAs once all MMAs issued so far have retired
__device__ __forceinline__ void wide_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(mx_map_to_rank(bar, 1)) : "memory");
}

// 16 neighbouring results of a row, `left` of them inside the matrix; `wide`: rows are multiples of 32 bytes and start on them
template <typename T>
__device__ __forceinline__ void store16(T* dst, const float (&v)[16], int left, bool wide) {
    if (wide && left >= 16) {
        constexpr int W = sizeof(T) == 4 ? 16 : 8;
        uint32_t w[W];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
        } else {
            union {
                T e[16];
                uint32_t u[8];
            } o;
#pragma unroll
            for (int i = 0; i < 16; ++i) o.e[i] = from_f32<T>(v[i]);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = o.u[i];
        }
#pragma unroll
        for (int i = 0; i < W; i += 8)
            st_global_32(reinterpret_cast<uint32_t*>(dst) + i, {w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5], w[i + 6], w[i + 7]});
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < left) dst[i] = from_f32<T>(v[i]);
    }
}

template <bool GATED>
__global__ void __launch_bounds__(kWideThreads, 1) mx4_wide_kernel(const WideParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ uint64_t bar_full[kWideStages];   // this CTA's stage has landed; leader: and the other CTA's
    __shared__ uint64_t bar_empty[kWideStages];  // the MMAs on the stage have retired
    __shared__ uint64_t bar_accum, bar_free;        // tile complete; leader: accumulator taken by all epilogue warps
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;

    const int tid = threadIdx.x, warp = mx_uniform_warp(), lane = tid & 31;
    const uint32_t crank = mx_cluster_rank();
    const int worker = (int)blockIdx.x / 2, workers = (int)gridDim.x / 2;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < kWideStages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), crank == 0 ? 2 : 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&bar_accum), 1);
        mbar_init(smem_u32(&bar_free), 16);
        fence_mbar_init();
    }
    if (warp == 1) {
        wide_alloc(smem_u32(&tmem_base_slot));
        grid_dep_launch();  // not before: see mx4_gemm.cu
    }
    tc_fence_before();
    __syncthreads();
    mx_cluster_sync();
    tc_fence_after();
    if (!p.early || warp != 0) grid_dep_wait();
    const uint32_t tmem_base = tmem_base_slot;

    // bar_empty, bar_accum and bar_free are arrived at by the pair's other CTA: commits of MMAs, and "accumulator taken". (Waits that acquire at the cluster's scope empty
    // the L1: with a bias 99 us for 86.) bar_full is in the first place a CTA's own copies.
    // A unit is two neighbouring activation tiles of one group (or its last one); an item is a unit x a 256-wide tile of weights.
    const int units = p.units ? (int)ld_l2_u32(p.n_units) : (p.M + 2 * kMxTileRows - 1) / (2 * kMxTileRows);
    const int items = units * p.w_tiles;
    constexpr int kGroup = 8;  // units whose items are neighbours: the operands of concurrent tiles are shared in the L2
    struct Item {
        int x_tile, w_tile, rows, expert, first;
    };
    auto item_of = [&](int i, Item& it) {
        int unit;
        if (p.units) {
            // An expert's items are neighbours, all its units on one tile of weights, then on the next: the weights come from HBM once, at an even rate.
            const uint4 run = ld_l2_u4(p.units + 2 * (i / p.w_tiles) + 1);
            const int in = i - (int)run.x * p.w_tiles;
            it.w_tile = in / (int)run.y;
            unit = (int)run.x + in - it.w_tile * (int)run.y;
        } else {
            const int per = kGroup * p.w_tiles, g = i / per, in = i - g * per, size = min(kGroup, units - g * kGroup);
            it.w_tile = in / size;
            unit = g * kGroup + in - it.w_tile * size;
        }
        it.x_tile = unit * 2 + (int)crank;
        it.expert = 0;
        it.first = it.x_tile * kMxTileRows;
        it.rows = p.M - it.first;
        if (p.units) {
            const uint4 u = ld_l2_u4(p.units + 2 * unit);
            it.expert = (int)u.x;
            it.first = (int)u.y + (int)crank * kMxTileRows;
            it.rows = (int)u.z - (int)crank * kMxTileRows;
            it.x_tile = (int)u.w + (int)crank;
        }
        it.rows = max(min(kMxTileRows, it.rows), 0);
    };

    int issued = 0;
    if (warp == 0) {
        int slot = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int i = worker; ok && i < items; i += workers) {
            Item it;
            item_of(i, it);
            // the last row tile of an odd number stands in for the one behind it, whose results are not stored
            const int t0 = GATED ? it.w_tile : 2 * it.w_tile, t1 = GATED ? it.w_tile : min(2 * it.w_tile + 1, p.row_tiles - 1);
            const uint8_t* w0 = p.W + (size_t)it.expert * p.w_expert_bytes + mx_tile_offset(t0, 0, p.k_tiles);
            const uint8_t* w1 = (GATED ? p.W_up : p.W) + (size_t)it.expert * p.w_expert_bytes + mx_tile_offset(t1, 0, p.k_tiles);
            const uint8_t* x = p.X + mx_tile_offset(it.x_tile, 0, p.k_tiles);
            const uint32_t x_bytes = (uint32_t)((it.rows + 7) & ~7) * 128u;
            // (a pair's second tile may lie behind the last: nothing of it is fetched, its rows of the accumulator are not used)
            const uint32_t bytes = (x_bytes ? x_bytes + kMxSfBytes : 0u) + kMxQBytes + 2 * kMxSfBytes;
            auto load_w = [&](int kt, uint32_t dst, uint32_t full) {
                const size_t at = (size_t)kt * kMxTileBytes;
                const uint32_t b = dst + kMxTileBytes;
                mbar_arrive_expect_tx(full, bytes);
                bulk_g2s(b, (crank ? w1 : w0) + at, kMxQBytes, full);
                bulk_g2s(b + kMxQBytes, w0 + at + kMxQBytes, kMxSfBytes, full);
                bulk_g2s(b + kMxQBytes + kMxSfBytes, w1 + at + kMxQBytes, kMxSfBytes, full);
            };
            auto load_x = [&](int kt, uint32_t dst, uint32_t full) {
                const uint8_t* src = x + (size_t)kt * kMxTileBytes;
                if (x_bytes == kMxQBytes) {
                    bulk_g2s(dst, src, kMxTileBytes, full);
                } else if (x_bytes) {
                    bulk_g2s(dst, src, x_bytes, full);
                    bulk_g2s(dst + kMxQBytes, src + kMxQBytes, kMxSfBytes, full);
                }
            };
            int kt = 0;
            if (i == worker) {  // the first stages' weights, then - behind the predecessor, whose results they are - the activations
                const int head = min(p.k_tiles, kWideStages);
                if (mx_elect())
                    for (int s = 0; s < head; ++s) load_w(s, sbase + s * kWideStageBytes, smem_u32(&bar_full[s]));
                __syncwarp();
                if (p.early) grid_dep_wait();
                if (mx_elect())
                    for (int s = 0; s < head; ++s) load_x(s, sbase + s * kWideStageBytes, smem_u32(&bar_full[s]));
                __syncwarp();
                issued = kt = head;
                slot = head == kWideStages ? 0 : head;
                if (slot == 0) phase ^= 1;
            }
            for (; kt < p.k_tiles; ++kt) {
                if (!(ok = mx_warp_wait<kMbarOrder>(smem_u32(&bar_empty[slot]), phase, &abort_flag, p.status, kDevTimeoutEmpty))) break;
                if (mx_elect()) {
                    load_w(kt, sbase + slot * kWideStageBytes, smem_u32(&bar_full[slot]));
                    load_x(kt, sbase + slot * kWideStageBytes, smem_u32(&bar_full[slot]));
                }
                __syncwarp();
                ++issued;
                if (++slot == kWideStages) { slot = 0; phase ^= 1; }
            }
        }
        if (p.early && worker >= items) grid_dep_wait();
    } else if (warp == 2) {
        if (crank == 1) {
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = worker; ok && i < items; i += workers)
                for (int kt = 0; kt < p.k_tiles; ++kt) {
                    if (!(ok = mx_warp_wait(smem_u32(&bar_full[slot]), phase, &abort_flag, p.status, kDevTimeoutFull))) break;
                    if (mx_elect()) mx_arrive_remote(mx_map_to_rank(smem_u32(&bar_full[slot]), 0));
                    __syncwarp();
                    if (++slot == kWideStages) { slot = 0; phase ^= 1; }
                }
        }
    } else if (warp == 1) {
        if (crank == 0) {
            int slot = 0;
            uint32_t phase = 0, free_phase = 1;
            const uint32_t id0 = instr_desc_mxf4(256, 256, 0), id2 = instr_desc_mxf4(256, 256, 2);
            bool ok = true;
            for (int i = worker; ok && i < items; i += workers) {
                if (!(ok = mx_warp_wait<kMbarOrder>(smem_u32(&bar_free), free_phase, &abort_flag, p.status, kDevTimeoutEmpty))) break;
                free_phase ^= 1;
                for (int kt = 0; kt < p.k_tiles; ++kt) {
                    if (!(ok = mx_warp_wait(smem_u32(&bar_full[slot]), phase, &abort_flag, p.status, kDevTimeoutFull))) break;
                    tc_fence_after();
                    const uint32_t a = sbase + slot * kWideStageBytes, b = a + kMxTileBytes, bs = b + kMxQBytes;
                    const uint32_t sf = tmem_base + 256u + (uint32_t)(slot * kWideSfCols);
                    const int left = p.K - kt * kMxTileK;
                    if (mx_elect()) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tmem_cp_scales<2>(sf + 4 * h, smem_desc_scales(a + kMxQBytes + 512 * h));
                            tmem_cp_scales<2>(sf + 8 + 8 * h, smem_desc_scales(bs + 512 * h));
                            tmem_cp_scales<2>(sf + 12 + 8 * h, smem_desc_scales(bs + kMxSfBytes + 512 * h));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (64 * j < left)
                                umma_mxf4<2>(tmem_base, smem_desc_sw128(a + 32 * j), smem_desc_sw128(b + 32 * j), j & 1 ? id2 : id0, sf + 4 * (j >> 1), sf + 8 + 8 * (j >> 1), (kt | j) != 0);
                        wide_commit(smem_u32(&bar_empty[slot]));
                        if (kt + 1 == p.k_tiles) wide_commit(smem_u32(&bar_accum));
                    }
                    __syncwarp();
                    if (++slot == kWideStages) { slot = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp >= kWideEpilogueWarp0) {
        const int half = (warp - kWideEpilogueWarp0) >> 2, r = (warp & 3) * 32 + lane;  // activation row of the tile = TMEM lane
        const uint32_t tlane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t free_bar = mx_map_to_rank(smem_u32(&bar_free), 0);
        const size_t elem = p.y_dtype == B200Q_DT_F32 ? 4 : 2;
        const bool wide = ((size_t)p.N * elem) % 32 == 0 && (reinterpret_cast<uintptr_t>(p.Y) & 31) == 0;
        uint32_t phase = 0;
        for (int i = worker; i < items; i += workers) {
            Item it;
            item_of(i, it);
            const int row = r < it.rows ? (p.units ? (int)ld_dep_u32(p.order + it.first + r) : it.first + r) : -1;
            if (!mx_warp_wait<kMbarOrder>(smem_u32(&bar_accum), phase, &abort_flag, p.status, kDevTimeoutMma)) break;
            phase ^= 1;
            tc_fence_after();
            // plain: columns 128 half ..; gated: gate columns 64 half .. in acc[0..63], up columns behind them
            uint32_t acc[8][16];
#pragma unroll
            for (int c = 0; c < 8; ++c) tmem_ld16(tlane + (uint32_t)(GATED ? (c < 4 ? 64 * half + 16 * c : 128 + 64 * half + 16 * (c - 4)) : 128 * half + 16 * c), acc[c]);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mx_arrive_remote(free_bar);
            const int n0 = GATED ? it.w_tile * 128 + 64 * half : it.w_tile * 256 + 128 * half;
            if (row >= 0) {
#pragma unroll
                for (int c = 0; c < (GATED ? 4 : 8); ++c) {
                    const int n = n0 + 16 * c;
                    if (n < p.N) {
                        float v[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            v[j] = __uint_as_float(acc[c][j]);
                            if constexpr (GATED) v[j] = silu_times(v[j], __uint_as_float(acc[4 + (c & 3)][j]));
                        }
                        if (!GATED && p.bias) {  // (value by value: 2000 x 14336 x 4096 takes 86 us with a bias, 49 without)
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (n + j < p.N) v[j] += load_bias(p.bias, p.bias_dtype, (size_t)it.expert * p.N + n + j);
                        }
                        const size_t o = (size_t)row * p.N + n;
                        if (p.y_dtype == B200Q_DT_F32) store16(static_cast<float*>(p.Y) + o, v, p.N - n, wide);
                        else if (p.y_dtype == B200Q_DT_F16) store16(static_cast<__half*>(p.Y) + o, v, p.N - n, wide);
                        else store16(static_cast<__nv_bfloat16*>(p.Y) + o, v, p.N - n, wide);
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) {  // given up: let the copies in flight land before the CTA's shared memory is given away
        for (int kt = max(issued - kWideStages, 0); kt < issued; ++kt)
            mbar_wait_bounded(smem_u32(&bar_full[kt % kWideStages]), (uint32_t)(kt / kWideStages) & 1u, p.status, kDevTimeoutFull, 1u << 12);
    }
    __syncwarp();
    mx_cluster_sync();  // nobody leaves while the pair's MMAs or arrivals may still reach it
    if (warp == 1) wide_dealloc(tmem_base);
}

template <bool GATED>
static int launch_wide(const WideParams& p, int64_t units, int sms, cudaStream_t st) {
    auto kern = mx4_wide_kernel<GATED>;
    constexpr int smem = kWideStages * kWideStageBytes + 1024;
    static bool configured[64] = {};
    int dev = 0;
    B200Q_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        B200Q_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int64_t items = units * p.w_tiles;
    if (items > (1LL << 30)) return fail(B200Q_ERR_UNSUPPORTED, "mx4: %lld tiles are more than one launch takes", (long long)items);
    const int workers = items < sms / 2 ? (int)items : sms / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(workers * 2));
    cfg.blockDim = dim3(kWideThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_option() >= 0 ? 2 : 1;
    B200Q_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return B200Q_OK;
}

// One matrix (plan == nullptr: M rows of X) or the experts of a plan (buffer laid out for `pairs` pairs and E experts).
int launch_mx4_wide(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                    int E, int early, int sms, int* status, cudaStream_t st) {
    WideParams p = {};
    p.early = early && pdl_option() >= 0;
    p.W = static_cast<const uint8_t*>(W);
    p.W_up = static_cast<const uint8_t*>(W_up);
    p.X = static_cast<const uint8_t*>(X);
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    p.Y = Y;
    p.y_dtype = y_dtype;
    p.status = status;
    p.M = M;
    p.N = N;
    p.K = K;
    p.k_tiles = mx_k_tiles(K);
    p.row_tiles = (int)mx_row_tiles(N);
    p.w_tiles = W_up ? p.row_tiles : (p.row_tiles + 1) / 2;
    int64_t units = (mx_row_tiles(M) + 1) / 2;
    if (plan) {
        const MoePlanLayout l = moe_plan_layout(pairs, E);
        p.w_expert_bytes = mx_image_bytes(N, K);
        p.units = reinterpret_cast<const int4*>(plan + l.units);
        p.n_units = plan + l.n_tiles + 1;
        p.order = plan + l.order;
        units = l.max_units;
    }
    return W_up ? launch_wide<true>(p, units, sms, st) : launch_wide<false>(p, units, sms, st);
}

}  // namespace b200q
