// Products of MXFP4 weights with few activation rows (decode): mx4_gemm.cu's arithmetic on 128 weight rows x 16 or 32
// activation rows, with the quantisation of the activations inside - the same values as b200q_mx4_quantize writes, kept in
// shared memory only. A projection is one launch, without a workspace.
//
// Bound by the weights' way from HBM (17 bits of 32 per weight); everything else has to hide behind it. A CTA has 128 rows and a share of the
// columns; its loader asks for the first stages at once while four warps quantise the CTA's part of the activations, one MMA step of 64 columns
// takes a few dozen clocks, and the shares of a cluster of up to eight CTAs meet through distributed shared memory in rank order.
//   warp 0  loader    warp 1  TMEM, MMAs    warps 2..5  quantisation, epilogue
#include "mx4_common.cuh"

namespace b200q {

constexpr int kFewQuantWarps = 8, kFewThreads = 64 + 32 * kFewQuantWarps, kFewMaxStages = 8, kFewRows = 32;

struct FewParams {
    const uint8_t* W;
    const uint8_t* W_up;
    const void* X;
    const void* bias;
    void* Y;
    int* status;
    size_t w_expert_bytes;
    const int4* tiles;   // grouped: {expert, first place, rows, 0}; nullptr: one matrix, M rows
    const int* n_tiles;
    const int* order;    // grouped: place -> pair, the row of Y
    int pairs_per_row;   // grouped: pairs that share a row of X (1: X has a row for each pair)
    int M, N, K;
    int k_tiles, split_log2, split_tiles;  // CTA rank r of a cluster of 2^split_log2 works on column tiles [r * split_tiles, ..)
    int bias_dtype, y_dtype;
    int n_cols;          // activation rows of the MMA, 16 or 32
    int n_stages;
    int experts;
    uint32_t tmem_cols;
};

template <int MATS, typename XT>
__global__ void __launch_bounds__(kFewThreads) mx4_few_kernel(const FewParams p) {
    constexpr uint32_t kStage = MATS * kMxTileBytes;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ uint64_t bar_full[kFewMaxStages], bar_empty[kFewMaxStages], bar_x, bar_accum, bar_parts;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ int pair_of[kFewRows];

    // Most of this kernel's time beside the weights' is latency, so what can be worked out ahead of a wait is, and nothing divides.
    const int tid = threadIdx.x, warp = mx_uniform_warp(), lane = tid & 31;
    const int split = 1 << p.split_log2, mine_log2 = 7 - p.split_log2, mine = 1 << mine_log2;
    const uint32_t crank = p.split_log2 ? mx_cluster_rank() : 0u;
    const int x_tile = (int)blockIdx.y, row_tile = (int)blockIdx.x >> p.split_log2;
    const int kt0 = (int)crank * p.split_tiles, share = max(min(p.split_tiles, p.k_tiles - kt0), 0);
    // [ring][activations: per column tile n_cols rows of 128 bytes, then 1024 bytes of scales][parts: see the epilogue]
    const uint32_t x_base = sbase + (uint32_t)p.n_stages * kStage, x_step = (uint32_t)p.n_cols * 128u + kMxSfBytes;
    const uint32_t parts = x_base + (uint32_t)p.split_tiles * x_step;
    const size_t w_at = mx_tile_offset(row_tile, kt0, p.k_tiles);

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < p.n_stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&bar_x), kFewQuantWarps);
        mbar_init(smem_u32(&bar_accum), 1);
        mbar_init(smem_u32(&bar_parts), 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), p.tmem_cols);
        tmem_relinquish();
    }
    grid_dep_launch();
    // The L2 hears about the weights while the predecessor still runs. Whose they are in a grouped product the plan says, which the predecessor
    // may be writing: a hint may be wrong, so it is only checked to lie inside the weights.
    if (warp == 0 && share > 0) {
        int e = 0;
        if (p.tiles) e = (unsigned)x_tile < ld_dep_u32(p.n_tiles) ? (int)ld_dep_u32(&p.tiles[x_tile].x) : -1;
        if ((unsigned)e < (unsigned)p.experts && mx_elect()) {
            const size_t at = (size_t)e * p.w_expert_bytes + w_at;
            bulk_prefetch_l2(p.W + at, (uint32_t)share * kMxTileBytes);
            if (MATS == 2) bulk_prefetch_l2(p.W_up + at, (uint32_t)share * kMxTileBytes);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (p.split_log2) mx_cluster_arrive();  // waited for before the first sums are sent: by then every CTA's barriers exist
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    grid_dep_wait();

    int rows = p.M, expert = 0, first = 0;
    if (p.tiles) {
        const int n_tiles = (int)ld_dep_u32(p.n_tiles);
        const uint4 t = ld_dep_u4(p.tiles + x_tile);  // (there is room for every x_tile of the grid)
        const bool mine_is = x_tile < n_tiles;
        expert = mine_is ? (int)t.x : 0;
        first = (int)t.y;
        rows = mine_is ? (int)t.z : 0;
    }
    const int n_kt = rows > 0 ? share : 0;
    int issued = 0;
    bool live = true;

    if (warp == 0) {
        const size_t at = (size_t)expert * p.w_expert_bytes + w_at;
        const uint8_t *w0 = p.W + at, *w1 = MATS == 2 ? p.W_up + at : nullptr;
        int slot = 0;
        uint32_t phase = 1;
        for (int kt = 0; kt < n_kt; ++kt) {
            if (!mx_warp_wait(smem_u32(&bar_empty[slot]), phase, &abort_flag, p.status, kDevTimeoutEmpty)) break;
            const uint32_t full = smem_u32(&bar_full[slot]), dst = sbase + slot * kStage;
            if (mx_elect()) {
                mbar_arrive_expect_tx(full, kStage);
                bulk_g2s(dst, w0, kMxTileBytes, full);
                if (MATS == 2) bulk_g2s(dst + kMxTileBytes, w1, kMxTileBytes, full);
            }
            __syncwarp();
            w0 += kMxTileBytes;
            if (MATS == 2) w1 += kMxTileBytes;
            ++issued;
            if (++slot == p.n_stages) { slot = 0; phase ^= 1; }
        }
    } else if (warp == 1) {
        int slot = 0;
        uint32_t phase = 0;
        const uint32_t id0 = instr_desc_mxf4(kMxTileRows, p.n_cols, 0), id2 = instr_desc_mxf4(kMxTileRows, p.n_cols, 2);
        if (n_kt > 0 && mx_warp_wait(smem_u32(&bar_x), 0, &abort_flag, p.status, kDevTimeoutFull)) {
            for (int kt = 0; kt < n_kt; ++kt) {
                if (!mx_warp_wait(smem_u32(&bar_full[slot]), phase, &abort_flag, p.status, kDevTimeoutFull)) break;
                tc_fence_after();
                const uint32_t st = sbase + slot * kStage, xs = x_base + (uint32_t)kt * x_step;
                const uint32_t sf = tmem_base + (uint32_t)(MATS * p.n_cols + slot * 8 * (MATS + 1));
                const int left = p.K - (kt0 + kt) * kMxTileK;
                if (mx_elect()) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m) tmem_cp_scales<1>(sf + 8 * m + 4 * h, smem_desc_scales(st + m * kMxTileBytes + kMxQBytes + 512 * h));
                        tmem_cp_scales<1>(sf + 8 * MATS + 4 * h, smem_desc_scales(xs + p.n_cols * 128 + 512 * h));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (64 * j < left) {
#pragma unroll
                            for (int m = 0; m < MATS; ++m)
                                umma_mxf4<1>(tmem_base + m * p.n_cols, smem_desc_sw128(st + m * kMxTileBytes + 32 * j), smem_desc_sw128(xs + 32 * j), j & 1 ? id2 : id0,
                                             sf + 8 * m + 4 * (j >> 1), sf + 8 * MATS + 4 * (j >> 1), (kt | j) != 0);
                        }
                    umma_commit(smem_u32(&bar_empty[slot]));
                    if (kt + 1 == n_kt) umma_commit(smem_u32(&bar_accum));
                }
                __syncwarp();
                if (++slot == p.n_stages) { slot = 0; phase ^= 1; }
            }
        }
    } else {
        // lane r: the pair (row of Y) of activation row r
        const int my_pair = p.tiles && lane < rows ? (int)ld_dep_u32(p.order + first + lane) : lane;
        const int my_src = p.pairs_per_row > 1 ? my_pair / p.pairs_per_row : my_pair;
        if (warp < 6) pair_of[lane] = my_pair;  // (the epilogue's warps, all the same values)
        if (n_kt > 0) {
            // A warp quantises 256 columns of a row at a time, lane 4 b + s elements 8 s .. 8 s + 7 of block b, with the next row's loads under way.
            // Up to eight column tiles the warps stand on one each, several rows abreast.
            const int b = lane >> 2, s = lane & 3, w = warp - 2;
            const int abreast = n_kt < kFewQuantWarps ? kFewQuantWarps / n_kt : 1, r0 = w / n_kt;
            if (r0 < abreast) {
                for (int kt = w - r0 * n_kt; kt < n_kt; kt += kFewQuantWarps) {
                    const int k = (kt0 + kt) * kMxTileK + 8 * lane;
                    const XT* x = static_cast<const XT*>(p.X) + k;
                    const uint32_t at = x_base + (uint32_t)kt * x_step, to = at + 4 * s, sc_to = at + (uint32_t)(p.n_cols * 128 + (lane >> 4) * 512);
                    float v[8], next[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = next[j] = 0.f;
                    int64_t src = __shfl_sync(0xffffffffu, my_src, r0 & 31);
                    if (r0 < rows && k < p.K) mx_load8(x + src * p.K, v);
                    for (int r = r0; r < rows; r += abreast) {
                        src = __shfl_sync(0xffffffffu, my_src, (r + abreast) & 31);
                        if (r + abreast < rows && k < p.K) mx_load8(x + src * p.K, next);
                        uint32_t sc;
                        const uint32_t q = mx_quantise8(v, sc);
                        uint32_t word = sc << (8 * (b & 3));
                        word |= __shfl_xor_sync(0xffffffffu, word, 4);
                        word |= __shfl_xor_sync(0xffffffffu, word, 8);
                        sts32(to + (uint32_t)(r >> 3) * 1024u + (uint32_t)(r & 7) * 128u + ((uint32_t)(b ^ (r & 7)) << 4), q);
                        if ((lane & 15) == 0) sts32(sc_to + (uint32_t)r * 16u, word);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = next[j];
                    }
                }
            }
            fence_proxy_async_smem();  // generic-proxy writes -> visible to the tensor cores
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_x));
        }
        __syncwarp();
    }
    if (warp >= 2 && warp < 6 && rows > 0) {  // epilogue, each warp its lane quarter
        const int r = (warp & 3) * 32 + lane;  // weight row of the tile = TMEM lane
        const uint32_t tlane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        if (p.split_log2 == 0) {
            const int my_pair = pair_of[lane];
            const int64_t n = (int64_t)row_tile * kMxTileRows + r;
            const float bv = p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, (size_t)expert * p.N + n) : 0.f;
            live = mx_warp_wait(smem_u32(&bar_accum), 0, &abort_flag, p.status, kDevTimeoutMma);
            tc_fence_after();
            for (int c = 0; c < rows; c += 16) {
                uint32_t a[MATS][16];
#pragma unroll
                for (int m = 0; m < MATS; ++m) tmem_ld16(tlane + (uint32_t)(m * p.n_cols + c), a[m]);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (c + j < rows) {
                        const size_t row = (size_t)__shfl_sync(0xffffffffu, my_pair, c + j);
                        float v = __uint_as_float(a[0][j]) + bv;
                        if (MATS == 2) v = silu_times(__uint_as_float(a[0][j]), __uint_as_float(a[MATS - 1][j]));
                        if (live && n < p.N) store_y(p.Y, p.y_dtype, row * p.N + n, v);
                    }
                }
            }
        } else {
            // Rank q adds up weight rows [q * mine, + mine) of the tile. Every rank sends it its sums of these - parts[rank][matrix][activation
            // row][mine], weight row r being row r % mine of rank r / mine - and its barrier counts the bytes.
            if (tid == 64) mbar_arrive_expect_tx(smem_u32(&bar_parts), (uint32_t)(MATS * rows) << 9);
            const uint32_t to_rank = (uint32_t)(r >> mine_log2);
            const uint32_t to = mx_map_to_rank(parts + (uint32_t)((((((int)crank * MATS * rows) << mine_log2)) + (r & (mine - 1))) * 4), to_rank);
            const uint32_t to_bar = mx_map_to_rank(smem_u32(&bar_parts), to_rank);
            const int t0 = (tid - 64) >> mine_log2;  // this thread's results: activation rows t0, t0 + split, .. of weight row x
            const int x = (tid - 64) & (mine - 1);
            const int64_t n = (int64_t)row_tile * kMxTileRows + (int)crank * mine + x;
            const float bv = p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, (size_t)expert * p.N + n) : 0.f;
            mx_cluster_wait();
            if (n_kt > 0) live = mx_warp_wait(smem_u32(&bar_accum), 0, &abort_flag, p.status, kDevTimeoutMma);
            tc_fence_after();
            for (int c = 0; c < rows; c += 16) {
                uint32_t a[MATS][16];
#pragma unroll
                for (int m = 0; m < MATS; ++m) tmem_ld16(tlane + (uint32_t)(m * p.n_cols + c), a[m]);
                tmem_ld_wait();
                // (a rank that has given up sends zeros: its peers come to an end, the status says that the result is void)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < rows) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m)
                            st_async_f32(to + ((uint32_t)(m * rows + c + j) << (mine_log2 + 2)), live && n_kt > 0 ? __uint_as_float(a[m][j]) : 0.f, to_bar);
                    }
            }
            const bool ok = mx_warp_wait(smem_u32(&bar_parts), 0, &abort_flag, p.status, kDevTimeoutPeer);
            if (ok && n < p.N) {
                for (int t = t0; t < rows; t += split) {
                    float s[MATS];
#pragma unroll
                    for (int m = 0; m < MATS; ++m) {
                        s[m] = 0.f;
                        for (int q = 0; q < split; ++q) s[m] += lds_f32(parts + (uint32_t)((((q * MATS + m) * rows + t) << mine_log2) + x) * 4u);
                    }
                    float v = s[0] + bv;
                    if (MATS == 2) v = silu_times(s[0], s[MATS - 1]);
                    store_y(p.Y, p.y_dtype, (size_t)pair_of[t] * p.N + n, v);
                }
            }
        }
    } else if (p.split_log2) {
        mx_cluster_wait();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) {  // given up: let the copies in flight land before the CTA's shared memory is given away
        for (int kt = max(issued - p.n_stages, 0); kt < issued; ++kt)
            mbar_wait_bounded(smem_u32(&bar_full[kt % p.n_stages]), (uint32_t)(kt / p.n_stages) & 1u, p.status, kDevTimeoutFull, 1u << 12);
    }
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

static int g_few_split = 0, g_few_budget = 0;

template <int MATS, typename XT>
static int launch_few(const FewParams& q, int64_t x_tiles, int sms, cudaStream_t st, bool* taken) {
    auto kern = mx4_few_kernel<MATS, XT>;
    FewParams p = q;
    constexpr int stage = MATS * kMxTileBytes;
    const int64_t row_tiles = mx_row_tiles(p.N), tiles = x_tiles * row_tiles;
    p.split_log2 = 0;
    while (p.split_log2 < 3 && tiles << (p.split_log2 + 1) <= 3 * sms && p.k_tiles >= 4 << p.split_log2) ++p.split_log2;
    if (g_few_split) p.split_log2 = g_few_split - 1;
    const int split = 1 << p.split_log2;
    p.split_tiles = (p.k_tiles + split - 1) / split;
    const size_t x_bytes = (size_t)p.split_tiles * (p.n_cols * 128 + kMxSfBytes), parts = split > 1 ? (size_t)MATS * p.n_cols * 512 : 0;
    *taken = false;
    if (x_bytes + parts > 64 * 1024 || tiles * split > 2147483647LL || x_tiles > 65535) return B200Q_OK;
    const int acc = MATS * p.n_cols, sf = 8 * (MATS + 1);
    int budget = MATS == 1 ? 74 * 1024 : 111 * 1024;
    if (g_few_budget) budget = g_few_budget * 1024;
    if ((int)(x_bytes + parts) + 3 * stage > budget) budget = 111 * 1024;
    if ((int)(x_bytes + parts) + 3 * stage > budget) budget = 222 * 1024;
    p.n_stages = (budget - (int)(x_bytes + parts)) / stage;
    if (p.n_stages > kFewMaxStages) p.n_stages = kFewMaxStages;
    if (p.n_stages > p.split_tiles) p.n_stages = p.split_tiles;
    while (acc + p.n_stages * sf > 256) --p.n_stages;
    p.tmem_cols = acc + p.n_stages * sf <= 128 ? 128u : 256u;
    size_t smem = (size_t)p.n_stages * stage + x_bytes + parts;
    static int static_smem[64] = {};
    int dev = 0;
    B200Q_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !static_smem[dev]) {
        B200Q_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024));
        cudaFuncAttributes a;
        B200Q_CUDA_TRY(cudaFuncGetAttributes(&a, kern));
        if (dev >= 0 && dev < 64) static_smem[dev] = (int)a.sharedSizeBytes;
    }
    smem = mx_smem_for_tmem(smem + 1024, p.tmem_cols);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(row_tiles * split), (unsigned)x_tiles);
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_option() >= 0 ? 2 : 1;
    *taken = true;
    B200Q_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return B200Q_OK;
}

// Y = X W^T for at most 32 rows of X (M of one matrix, or the pairs of a plan: no group can be larger). X is dense, of x_dtype.
// `taken` says whether the shape is one of the kernel's.
int launch_mx4_few(const void* W, const void* W_up, const void* X, int x_dtype, const void* bias, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                   int pairs_per_row, int E, int sms, int* status, cudaStream_t st, bool* taken) {
    FewParams p = {};
    p.W = static_cast<const uint8_t*>(W);
    p.W_up = static_cast<const uint8_t*>(W_up);
    p.X = X;
    p.bias = bias;
    p.bias_dtype = x_dtype;
    p.Y = Y;
    p.y_dtype = y_dtype;
    p.status = status;
    p.M = M;
    p.N = N;
    p.K = K;
    p.k_tiles = mx_k_tiles(K);
    p.pairs_per_row = pairs_per_row;
    p.experts = plan ? E : 1;
    int64_t x_tiles = 1, rows = M;
    if (plan) {
        const MoePlanLayout l = moe_plan_layout(pairs, E);
        p.w_expert_bytes = mx_image_bytes(N, K);
        p.tiles = reinterpret_cast<const int4*>(plan + l.tiles);
        p.n_tiles = plan + l.n_tiles;
        p.order = plan + l.order;
        x_tiles = l.max_tiles;
        rows = pairs;
    }
    *taken = false;
    if (rows > 32) return B200Q_OK;
    p.n_cols = rows > 16 ? 32 : 16;
    auto run = [&](auto zero) {
        using XT = decltype(zero);
        return W_up ? launch_few<2, XT>(p, x_tiles, sms, st, taken) : launch_few<1, XT>(p, x_tiles, sms, st, taken);
    };
    return x_dtype == B200Q_DT_F32 ? run(0.f) : x_dtype == B200Q_DT_F16 ? run(__half()) : run(__nv_bfloat16());
}

void few_set(int split, int budget) { g_few_split = split; g_few_budget = budget; }

}  // namespace b200q
