// Products of MXFP4 images on the block-scaled tensor cores (tcgen05 kind::mxf4):
//   Y(M,N) = X(M,K) W(N,K)^T (+ bias),  both operands E2M1 with one E8M0 scale per 32 columns, FP32 accumulation in TMEM,
// for one matrix (a projection) or, over the tiles of a MoePlan, for the matrices of many experts; with two matrices the
// result is silu(gate) * up.
//
// A CTA owns 128 weight rows (the MMA's M, TMEM lanes) and up to 128 activation rows (its N, TMEM columns), so that a
// product of a few rows wastes little and results of one activation row leave as contiguous stores. Per 256 columns a
// stage holds one tile of each image - one bulk copy each, scales included - and costs two tcgen05.cp per operand (128
// columns' scales to TMEM) and four MMAs of 64 columns. Products and sums are exact or FP32: the operands need no decoding.
//   warp 0      one thread streams the stages through the ring
//   warp 1      TMEM allocation; one thread issues copies of scales, MMAs and commits
//   warps 2..5  epilogue (each its lane quarter)
// Few tiles: the k range is cut over the CTAs of a cluster of up to eight, whose partial sums meet through distributed
// shared memory in rank order - no workspace, no atomics, the same result on every run.
// All waits are bounded as in the other kernels; on a timeout the CTA records a status code, still takes part in the
// cluster barriers, frees its TMEM and returns.
#include "mx4_common.cuh"

namespace b200q {

constexpr int kMxThreads = 192, kMxEpilogueWarp0 = 2;
constexpr int kMxMaxStages = 12;

struct MxParams {
    const uint8_t* W;      // image of the (gate) weights; expert e's lies e * w_expert_bytes behind
    const uint8_t* W_up;   // image of the up weights, or nullptr
    const uint8_t* X;      // image of the activations
    const void* bias;      // N values (per expert), or nullptr
    void* Y;
    int* status;
    size_t w_expert_bytes;
    const int4* tiles;     // grouped: {expert, first place, rows, 0} of each tile of X; nullptr: one matrix, M rows
    const int* n_tiles;
    const int* order;      // grouped: place -> row of Y
    int M, N, K;
    int row_tiles, k_tiles, split, split_tiles;  // CTA rank r of a cluster of `split` works on k tiles [r * split_tiles, ..)
    int bias_dtype, y_dtype;
    int n_cols;            // accumulator columns per matrix (activation rows of a full tile, a multiple of 16)
    int n_stages, stage_bytes;
    uint32_t tmem_cols;
};

template <int MATS>  // weight matrices: 1, or 2 for silu(gate) * up
__global__ void __launch_bounds__(kMxThreads) mx4_gemm_kernel(const MxParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ uint64_t bar_full[kMxMaxStages], bar_empty[kMxMaxStages], bar_accum;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ int out_row[kMxTileRows];  // row of Y of each activation row of the tile

    const int tid = threadIdx.x, warp = mx_uniform_warp(), lane = tid & 31;
    const uint32_t crank = p.split > 1 ? mx_cluster_rank() : 0u;
    const int64_t work = (int64_t)(blockIdx.x / (unsigned)p.split);
    const int64_t x_tile = work / p.row_tiles;
    const int row_tile = (int)(work - x_tile * p.row_tiles);

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < p.n_stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&bar_accum), 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), p.tmem_cols);
        tmem_relinquish();
    }
    grid_dep_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dep_wait();
    const uint32_t tmem_base = tmem_base_slot;

    // what this CTA works on; the same for all CTAs of a cluster
    int rows, expert = 0, first = 0;
    if (p.tiles) {
        rows = 0;
        if (x_tile < (int64_t)(int)ld_dep_u32(p.n_tiles)) {
            const uint4 t = ld_dep_u4(p.tiles + x_tile);
            expert = (int)t.x;
            first = (int)t.y;
            rows = (int)t.z;
        }
        for (int i = tid; i < rows; i += kMxThreads) out_row[i] = (int)ld_dep_u32(p.order + first + i);
    } else {
        rows = (int)min((int64_t)kMxTileRows, (int64_t)p.M - x_tile * kMxTileRows);
        for (int i = tid; i < rows; i += kMxThreads) out_row[i] = (int)(x_tile * kMxTileRows) + i;
    }
    __syncthreads();
    const int kt0 = (int)crank * p.split_tiles, n_kt = rows > 0 ? min(p.split_tiles, p.k_tiles - kt0) : 0;
    const int n_mma = (rows + 15) & ~15;
    int issued = 0;  // warp 0's thread: stages requested

    const uint32_t sf_col0 = (uint32_t)(MATS * p.n_cols);  // scales behind the accumulators: per stage 8 columns for each matrix, 8 for X
    if (warp == 0) {
        const uint8_t* w0 = p.W + (size_t)expert * p.w_expert_bytes + mx_tile_offset(row_tile, kt0, p.k_tiles);
        const uint8_t* w1 = MATS == 2 ? p.W_up + (size_t)expert * p.w_expert_bytes + mx_tile_offset(row_tile, kt0, p.k_tiles) : nullptr;
        const uint8_t* x = p.X + mx_tile_offset(x_tile, kt0, p.k_tiles);
        const uint32_t x_bytes = (uint32_t)n_mma * 128u;
        int slot = 0;
        uint32_t phase = 1;
        for (int kt = 0; kt < n_kt; ++kt) {
            if (!mx_warp_wait(smem_u32(&bar_empty[slot]), phase, &abort_flag, p.status, kDevTimeoutEmpty)) break;
            const uint32_t full = smem_u32(&bar_full[slot]), dst = sbase + slot * p.stage_bytes;
            if (mx_elect()) {
                mbar_arrive_expect_tx(full, MATS * kMxTileBytes + x_bytes + kMxSfBytes);
                bulk_g2s(dst, w0, kMxTileBytes, full);
                if (MATS == 2) bulk_g2s(dst + kMxTileBytes, w1, kMxTileBytes, full);
                bulk_g2s(dst + MATS * kMxTileBytes + kMxSfBytes, x, x_bytes, full);
                bulk_g2s(dst + MATS * kMxTileBytes, x + kMxQBytes, kMxSfBytes, full);
            }
            __syncwarp();
            w0 += kMxTileBytes;
            if (MATS == 2) w1 += kMxTileBytes;
            x += kMxTileBytes;
            ++issued;
            if (++slot == p.n_stages) { slot = 0; phase ^= 1; }
        }
    } else if (warp == 1) {
        int slot = 0;
        uint32_t phase = 0;
        const uint32_t id0 = instr_desc_mxf4(kMxTileRows, n_mma, 0), id2 = instr_desc_mxf4(kMxTileRows, n_mma, 2);
        for (int kt = 0; kt < n_kt; ++kt) {
            if (!mx_warp_wait(smem_u32(&bar_full[slot]), phase, &abort_flag, p.status, kDevTimeoutFull)) break;
            tc_fence_after();
            const uint32_t st = sbase + slot * p.stage_bytes, xs = st + MATS * kMxTileBytes;
            const uint32_t sf = tmem_base + sf_col0 + (uint32_t)(slot * 8 * (MATS + 1));
            const int left = p.K - (kt0 + kt) * kMxTileK;  // columns beyond K are zeros: whole steps of them are left out
            if (mx_elect()) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int m = 0; m < MATS; ++m) tmem_cp_scales<1>(sf + 8 * m + 4 * h, smem_desc_scales(st + m * kMxTileBytes + kMxQBytes + 512 * h));
                    tmem_cp_scales<1>(sf + 8 * MATS + 4 * h, smem_desc_scales(xs + 512 * h));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (64 * j < left) {
                        const uint64_t xd = smem_desc_sw128(xs + kMxSfBytes + 32 * j);
#pragma unroll
                        for (int m = 0; m < MATS; ++m)
                            umma_mxf4<1>(tmem_base + m * p.n_cols, smem_desc_sw128(st + m * kMxTileBytes + 32 * j), xd, j & 1 ? id2 : id0,
                                         sf + 8 * m + 4 * (j >> 1), sf + 8 * MATS + 4 * (j >> 1), (kt | j) != 0);
                    }
                }
                umma_commit(smem_u32(&bar_empty[slot]));
            }
            __syncwarp();
            if (++slot == p.n_stages) { slot = 0; phase ^= 1; }
        }
        if (rows > 0 && mx_elect()) umma_commit(smem_u32(&bar_accum));
        __syncwarp();
    }
    // ---- epilogue
    bool live = true;
    if (warp >= kMxEpilogueWarp0) {
        if (rows > 0) live = mx_warp_wait(smem_u32(&bar_accum), 0, &abort_flag, p.status, kDevTimeoutMma);
        tc_fence_after();
        const int r = (warp & 3) * 32 + lane;  // weight row of the tile = TMEM lane
        const uint32_t tlane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const int64_t n = (int64_t)row_tile * kMxTileRows + r;
        if (live && rows > 0 && p.split == 1) {
            const float bv = p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, (size_t)expert * p.N + n) : 0.f;
            for (int c = 0; c < n_mma; c += 16) {
                uint32_t a[16], b[16];
                tmem_ld16(tlane + (uint32_t)c, a);
                if (MATS == 2) tmem_ld16(tlane + (uint32_t)(p.n_cols + c), b);
                tmem_ld_wait();
                if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (c + j < rows) {
                            float v = __uint_as_float(a[j]) + bv;
                            if (MATS == 2) v = silu_times(__uint_as_float(a[j]), __uint_as_float(b[j]));
                            store_y(p.Y, p.y_dtype, (size_t)out_row[c + j] * p.N + n, v);
                        }
                    }
                }
            }
        } else if (rows > 0 && p.split > 1) {
            // partial sums [matrix][activation row][128] over the ring, whose stages are all consumed
            float* part = reinterpret_cast<float*>(smem_raw + (sbase - smem_u32(smem_raw)));
            for (int m = 0; m < MATS; ++m)
                for (int c = 0; c < n_mma; c += 16) {
                    uint32_t a[16];
                    tmem_ld16(tlane + (uint32_t)(m * p.n_cols + c), a);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < rows) part[(m * p.n_cols + c + j) * 128 + r] = live && n_kt > 0 ? __uint_as_float(a[j]) : 0.f;
                }
        }
    }
    if (p.split > 1) {
        mx_cluster_sync();
        // rank q adds up weight rows [q * 128 / split, ..) of the tile, ranks in order
        const int mine = kMxTileRows / p.split;
        if (live && rows > 0) {
            for (int i = tid; i < rows * mine; i += kMxThreads) {
                const int t = i / mine, r = (int)crank * mine + (i - t * mine);
                const int64_t n = (int64_t)row_tile * kMxTileRows + r;
                if (n >= p.N) continue;
                float s[MATS];
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    s[m] = 0.f;
                    const uint32_t at = sbase + (uint32_t)(((m * p.n_cols + t) * 128 + r) * 4);
                    for (int q = 0; q < p.split; ++q) s[m] += ld_cluster_f32(mx_map_to_rank(at, (uint32_t)q));
                }
                float v = s[0] + (p.bias ? load_bias(p.bias, p.bias_dtype, (size_t)expert * p.N + n) : 0.f);
                if (MATS == 2) v = silu_times(s[0], s[MATS - 1]);
                store_y(p.Y, p.y_dtype, (size_t)out_row[t] * p.N + n, v);
            }
        }
        mx_cluster_sync();  // nobody leaves while its partial sums are read
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) {  // given up: let the copies in flight land before the CTA's shared memory is given away
        for (int kt = max(issued - p.n_stages, 0); kt < issued; ++kt)
            mbar_wait_bounded(smem_u32(&bar_full[kt % p.n_stages]), (uint32_t)(kt / p.n_stages) & 1u, p.status, kDevTimeoutFull, 1u << 12);
    }
    if (warp == 1) tmem_dealloc(tmem_base, p.tmem_cols);
}

template <int MATS>
static int launch_mx_gemm(const MxParams& p, int64_t x_tiles, size_t smem, cudaStream_t st) {
    auto kern = mx4_gemm_kernel<MATS>;
    static bool configured[64] = {};
    int dev = 0;
    B200Q_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        B200Q_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int64_t blocks = x_tiles * p.row_tiles * p.split;
    if (blocks > 2147483647LL) return fail(B200Q_ERR_UNSUPPORTED, "mx4: %lld blocks are more than a grid holds", (long long)blocks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kMxThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_option() >= 0 ? 2 : 1;
    B200Q_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return B200Q_OK;
}

int launch_mx4_wide(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                    int E, int sms, int* status, cudaStream_t st);

static int g_mx4_wide = 1;
void mx4_set_wide(int v) { g_mx4_wide = v; }
int mx4_get_wide() { return g_mx4_wide; }
static int g_mx4_few = 32;
void mx4_set_few(int v) { g_mx4_few = v; }
int mx4_get_few() { return g_mx4_few; }

// One matrix (plan == nullptr: M rows of X) or the experts of a plan (buffer laid out for `pairs` pairs and E experts).
int launch_mx4_gemm(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K,
                    const int* plan, int64_t pairs, int E, int sms, int* status, cudaStream_t st) {
    const bool many = plan ? pairs >= 64LL * E : M >= 192;
    if (g_mx4_wide == 2 || (g_mx4_wide == 1 && many))
        return launch_mx4_wide(W, W_up, X, bias, bias_dtype, Y, y_dtype, M, N, K, plan, pairs, E, sms, status, st);
    MxParams p = {};
    const int mats = W_up ? 2 : 1;
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
    int64_t x_tiles = mx_row_tiles(M), rows_most = M;
    if (plan) {
        const MoePlanLayout l = moe_plan_layout(pairs, E);
        p.w_expert_bytes = mx_image_bytes(N, K);
        p.tiles = reinterpret_cast<const int4*>(plan + l.tiles);
        p.n_tiles = plan + l.n_tiles;
        p.order = plan + l.order;
        x_tiles = l.max_tiles;
        rows_most = pairs;
    }
    p.n_cols = rows_most >= kMxTileRows ? kMxTileRows : (int)((rows_most + 15) & ~15);
    p.stage_bytes = mats * kMxTileBytes + kMxSfBytes + p.n_cols * 128;
    // Split K while the CTAs do not fill the SMs twice and every share keeps two tiles or more.
    p.split = 1;
    while (p.split < 8 && x_tiles * p.row_tiles * p.split * 2 <= 2 * sms && p.k_tiles >= 4 * p.split) p.split *= 2;
    p.split_tiles = (p.k_tiles + p.split - 1) / p.split;
    // Two CTAs share an SM where 256 TMEM columns do (accumulators and the stages' scales), else one has it alone. Shared memory is
    // asked for such that TMEM cannot run out: CTAs that fit an SM by their shared memory fit its 512 columns too.
    const int acc = mats * p.n_cols, sf = 8 * (mats + 1);
    const bool two = acc + 4 * sf <= 256;
    const int budget = two ? 110 * 1024 : 222 * 1024;
    p.n_stages = budget / p.stage_bytes;
    if (p.n_stages > kMxMaxStages) p.n_stages = kMxMaxStages;
    const int cols = two ? 256 : 512;
    while (acc + p.n_stages * sf > cols) --p.n_stages;
    p.tmem_cols = (uint32_t)cols;
    size_t smem = (size_t)p.n_stages * p.stage_bytes;
    const size_t parts = p.split > 1 ? (size_t)mats * p.n_cols * 512 : 0;
    if (smem < parts) smem = parts;
    smem = mx_smem_for_tmem(smem + 1024, two ? 256 : 512);
    return mats == 2 ? launch_mx_gemm<2>(p, x_tiles, smem, st) : launch_mx_gemm<1>(p, x_tiles, smem, st);
}

}  // namespace b200q
