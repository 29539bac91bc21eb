// Products of MXFP4 images on the block-scaled tensor cores (tcgen05 kind::mxf4):
//   Y(M,N) = X(M,K) W(N,K)^T (+ bias),  both operands E2M1 with one E8M0 scale per 32 columns, FP32 accumulation in TMEM,
// for one matrix (a projection) or, over the tiles of a MoePlan, for the matrices of many experts; with two matrices the
// result is silu(gate) * up. This kernel is for few activation rows (mx4_wide.cu: many).
//
// A CTA owns 128 weight rows (the MMA's M, TMEM lanes) and up to 128 activation rows (its N, TMEM columns), so that a
// product of a few rows wastes little. Per 256 columns a stage holds one tile of each image - one bulk copy each, scales included -
// and costs two tcgen05.cp per operand (128 columns' scales to TMEM) and four MMAs of 64 columns. Nothing is decoded.
// Bound by the weights' way from HBM (17 bits of 32 per weight); everything else has to hide behind it.
//   warp 0       loader    warp 1  TMEM, scales, MMAs    warps 2..5  epilogue (each its lane quarter)
//
// XT = void: X is an image (mx4_quant.cu has made it just before). Otherwise X is dense, of at most 16 rows (decode), and warps 2..9 quantise the CTA's
// part of it first - the same values, kept in shared memory only: a projection is one launch, without a workspace.
//
// Few tiles: the k range is cut over the CTAs of a cluster of up to eight. Each rank sends its sums of a slice of the weight rows to the rank
// that adds the slice up, in rank order - no workspace, no atomics, the same result on every run. (With the sums fetched from the
// others' shared memory between two cluster barriers a launch took 1.5 us more.)
//
// All waits are bounded as in the other kernels; on a timeout the CTA records a status code, sends zeros, frees its TMEM and returns.
#include <atomic>
#include <type_traits>

#include "mx4_common.cuh"

namespace b200q {

// Dense X of up to kMxDenseRows rows. One row is well inside the weights' time, many are not: a warp quantises its rows one after the other while the full ring waits (14336 x 4096 at
// 1 / 8 / 16 rows 8.2 / 12.9 / 17.7 us, and 11.6 at 17, in two launches; 6400 x 8192 9.9 / 12.5 / 16.3 and 10.4; 1024 x 14336 at 8 rows 8.9).
constexpr int kMxMaxStages = 12, kMxDenseRows = 16;
constexpr int kMxDenseTiles = 32;  // dense X: most column tiles of a CTA (activations 96 KB, beside three gated stages 105 KB)
constexpr int kMxQuantWarps = 8;  // dense X: warps that quantise (four of them then have the epilogue)
template <typename XT>
constexpr bool kIsImage = std::is_same_v<XT, void>;
template <typename XT>
constexpr int kMxThreads = 64 + 32 * (kIsImage<XT> ? 4 : kMxQuantWarps);

struct MxParams {
    const uint8_t* W;
    const uint8_t* W_up;
    const void* X;         // image or dense rows
    const void* bias;      // N values (per expert), or nullptr
    void* Y;
    int* status;
    size_t w_expert_bytes;
    const int4* tiles;   // grouped: {expert, first place, rows, first pair}; nullptr: one matrix, M rows
    const int* n_tiles;
    const int* order;    // grouped: place -> pair, the row of Y
    int pairs_per_row;   // grouped, dense X: pairs that share a row of X (1: X has a row for each pair)
    int M, N, K;
    int x_tiles, row_tiles;  // tiles of activations (grouped: room for so many) and of 128 weight rows
    int k_tiles, split_log2, split_tiles;  // CTA rank r of a cluster of 2^split_log2 works on column tiles [r * split_tiles, ..)
    int bias_dtype, y_dtype;
    int n_cols;          // accumulator columns of a matrix: activation rows of the largest item, a multiple of 16
    int few_rows, n_stages, stage_bytes;  // the ring for items of up to few_rows activation rows,
    int big_stages, big_bytes;            // and in the same memory for those of more
    int experts;
    int early;           // the predecessor writes neither weights nor plan (it is the quantisation): they are read ahead of its end
    uint32_t tmem_cols;
};

template <int MATS, typename XT>
__global__ void __launch_bounds__(kMxThreads<XT>, kIsImage<XT> ? 2 : 3) mx4_gemm_kernel(const MxParams p) {
    constexpr uint32_t kWBytes = MATS * kMxTileBytes;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ uint64_t bar_full[kMxMaxStages], bar_empty[kMxMaxStages], bar_x, bar_accum, bar_free, bar_parts;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ int row_of[kMxTileRows];  // split: row of Y of each activation row of the tile

    // Much of this kernel's time beside the weights' is latency, so what can be worked out ahead of a wait is, and little divides.
    const int tid = threadIdx.x, warp = mx_uniform_warp(), lane = tid & 31;
    const int split = 1 << p.split_log2, mine_log2 = 7 - p.split_log2, mine = 1 << mine_log2;
    const uint32_t crank = p.split_log2 ? mx_cluster_rank() : 0u;
    const int kt0 = (int)crank * p.split_tiles, n_kt = max(min(p.split_tiles, p.k_tiles - kt0), 0);
    const int item0 = (int)blockIdx.x >> p.split_log2, item_step = (int)gridDim.x >> p.split_log2;
    // The activations of a column tile: 1024 bytes of scales, n_cols rows of 128 bytes. An image's are part of the stage; dense ones lie
    // behind the ring for all of the CTA's column tiles. Last the parts: see the epilogue.
    const uint32_t x_step = (uint32_t)p.n_cols * 128u + kMxSfBytes, x_base = sbase + (uint32_t)(p.n_stages * p.stage_bytes);
    const uint32_t parts = x_base + (kIsImage<XT> ? 0u : (uint32_t)p.split_tiles * x_step);

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < p.n_stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        if (!kIsImage<XT>) mbar_init(smem_u32(&bar_x), kMxQuantWarps);
        mbar_init(smem_u32(&bar_accum), 1);
        mbar_init(smem_u32(&bar_free), 4);
        mbar_init(smem_u32(&bar_parts), 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), p.tmem_cols);
        tmem_relinquish();
        grid_dep_launch();  // not before: a dependent that had taken the columns would wait for this CTA, and this CTA for the columns
    }
    // The L2 hears about the first weights while the predecessor still runs. Whose they are in a grouped product the plan says, which the predecessor
    // may be writing: a hint may be wrong, so it is only checked to lie inside the weights.
    if (warp == 0 && n_kt > 0 && !p.early) {
        const int x_tile = item0 / p.row_tiles;
        int e = 0;
        if (p.tiles) e = (unsigned)x_tile < ld_l2_u32(p.n_tiles) ? (int)ld_l2_u32(&p.tiles[x_tile].x) : -1;
        if ((unsigned)e < (unsigned)p.experts && mx_elect()) {
            const size_t at = (size_t)e * p.w_expert_bytes + mx_tile_offset(item0 - x_tile * p.row_tiles, kt0, p.k_tiles);
            bulk_prefetch_l2(p.W + at, (uint32_t)n_kt * kMxTileBytes);
            if (MATS == 2) bulk_prefetch_l2(p.W_up + at, (uint32_t)n_kt * kMxTileBytes);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (p.split_log2) mx_cluster_arrive();  // waited for before the first sums are sent: by then every CTA's barriers exist
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    if (!p.early || warp != 0) grid_dep_wait();

    // An item is a tile of activations x 128 weight rows. The ring's stages are laid out for `few_rows` activation rows, which the groups of a product
    // that comes here hardly ever exceed; an item of more has larger and fewer stages, and the ring runs empty before the layout changes.
    // (Waits go by one parity bit per slot, so that slots may be used in any order.)
    struct Item {
        int x_tile, row_tile, rows, expert, first, pair0;
    };
    const int n_items = (p.tiles ? min((int)ld_l2_u32(p.n_tiles), p.x_tiles) : p.x_tiles) * p.row_tiles;
    auto item_of = [&](int i, Item& it) {
        it.x_tile = i / p.row_tiles;
        it.row_tile = i - it.x_tile * p.row_tiles;
        it.expert = it.pair0 = 0;
        it.first = it.x_tile * kMxTileRows;
        it.rows = min(p.M - it.first, kMxTileRows);
        if (p.tiles) {
            const uint4 t = ld_l2_u4(p.tiles + it.x_tile);
            it.expert = (int)t.x;
            it.first = (int)t.y;
            it.rows = (int)t.z;
            it.pair0 = (int)t.w;
        }
    };
    auto stage_bytes_of = [&](int rows) { return rows > p.few_rows ? p.big_bytes : p.stage_bytes; };
    auto stages_of = [&](int rows) { return rows > p.few_rows ? p.big_stages : p.n_stages; };
    uint32_t parity = 0, used = 0;  // warp 0: parity of the next wait for each slot to be empty (= of its last fill); slots that have been filled

    if (warp == 0) {
        int slot = 0, stages = p.n_stages;
        parity = 0xffffffffu;
        bool ok = true;
        for (int i = item0; ok && i < n_items; i += item_step) {
            Item it;
            item_of(i, it);
            const size_t at = (size_t)it.expert * p.w_expert_bytes + mx_tile_offset(it.row_tile, kt0, p.k_tiles);
            const uint8_t *w0 = p.W + at, *w1 = MATS == 2 ? p.W_up + at : nullptr;
            const uint8_t* x = kIsImage<XT> ? static_cast<const uint8_t*>(p.X) + mx_tile_offset(it.x_tile, kt0, p.k_tiles) : nullptr;
            const uint32_t x_bytes = (uint32_t)((it.rows + 15) & ~15) * 128u, stage = (uint32_t)stage_bytes_of(it.rows);
            auto load_w = [&](int kt, int s) {
                const uint32_t dst = sbase + (uint32_t)s * stage, full = smem_u32(&bar_full[s]);
                mbar_arrive_expect_tx(full, kWBytes + (kIsImage<XT> ? x_bytes + kMxSfBytes : 0u));
                bulk_g2s(dst, w0 + (size_t)kt * kMxTileBytes, kMxTileBytes, full);
                if (MATS == 2) bulk_g2s(dst + kMxTileBytes, w1 + (size_t)kt * kMxTileBytes, kMxTileBytes, full);
            };
            auto load_x = [&](int kt, int s) {
                if constexpr (kIsImage<XT>) {
                    const uint32_t dst = sbase + (uint32_t)s * stage, full = smem_u32(&bar_full[s]);
                    const uint8_t* src = x + (size_t)kt * kMxTileBytes;
                    bulk_g2s(dst + kWBytes + kMxSfBytes, src, x_bytes, full);
                    bulk_g2s(dst + kWBytes, src + kMxQBytes, kMxSfBytes, full);
                }
            };
            int kt = 0;
            if (!used) {  // the first stages' weights, then - behind the predecessor, whose results they are - the activations
                stages = stages_of(it.rows);
                const int head = min(n_kt, stages);
                if (mx_elect())
                    for (int s = 0; s < head; ++s) load_w(s, s);
                __syncwarp();
                if (p.early) grid_dep_wait();
                if (kIsImage<XT> && mx_elect())
                    for (int s = 0; s < head; ++s) load_x(s, s);
                __syncwarp();
                kt = head;
                used = (1u << head) - 1u;
                parity ^= used;
                slot = head == stages ? 0 : head;
            } else if (stages != stages_of(it.rows)) {
                const int last = (slot ? slot : stages) - 1;
                if (!(ok = mx_warp_wait(smem_u32(&bar_empty[last]), parity >> last & 1u, &abort_flag, p.status, kDevTimeoutEmpty))) break;
                stages = stages_of(it.rows);
                slot = 0;
            }
            for (; kt < n_kt; ++kt) {
                if (!(ok = mx_warp_wait(smem_u32(&bar_empty[slot]), parity >> slot & 1u, &abort_flag, p.status, kDevTimeoutEmpty))) break;
                if (mx_elect()) {
                    load_w(kt, slot);
                    load_x(kt, slot);
                }
                __syncwarp();
                parity ^= 1u << slot;
                used |= 1u << slot;
                if (++slot == stages) slot = 0;
            }
        }
        if (p.early && !used) grid_dep_wait();
    } else if (warp == 1) {
        int slot = 0, stages = p.n_stages;
        uint32_t full_parity = 0, free_phase = 1;
        bool ok = true;
        for (int i = item0; ok && n_kt > 0 && i < n_items; i += item_step) {
            Item it;
            item_of(i, it);
            const int n_mma = kIsImage<XT> ? (it.rows + 15) & ~15 : kMxDenseRows;
            const uint32_t id0 = instr_desc_mxf4(kMxTileRows, n_mma, 0), id2 = instr_desc_mxf4(kMxTileRows, n_mma, 2), stage = (uint32_t)stage_bytes_of(it.rows);
            if (stages != stages_of(it.rows)) {
                stages = stages_of(it.rows);
                slot = 0;
            }
            if (!(ok = mx_warp_wait(smem_u32(&bar_free), free_phase, &abort_flag, p.status, kDevTimeoutEmpty))) break;
            free_phase ^= 1;
            if (!kIsImage<XT> && !(ok = mx_warp_wait(smem_u32(&bar_x), 0, &abort_flag, p.status, kDevTimeoutFull))) break;
            for (int kt = 0; kt < n_kt; ++kt) {
                if (!(ok = mx_warp_wait(smem_u32(&bar_full[slot]), full_parity >> slot & 1u, &abort_flag, p.status, kDevTimeoutFull))) break;
                full_parity ^= 1u << slot;
                tc_fence_after();
                const uint32_t st = sbase + (uint32_t)slot * stage, xs = kIsImage<XT> ? st + kWBytes : x_base + (uint32_t)kt * x_step;
                const uint32_t sf = tmem_base + (uint32_t)(MATS * p.n_cols + slot * 8 * (MATS + 1));
                const int left = p.K - (kt0 + kt) * kMxTileK;  // columns beyond K are zeros: whole steps of them are left out
                if (mx_elect()) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int m = 0; m < MATS; ++m) tmem_cp_scales<1>(sf + 8 * m + 4 * h, smem_desc_scales(st + m * kMxTileBytes + kMxQBytes + 512 * h));
                        tmem_cp_scales<1>(sf + 8 * MATS + 4 * h, smem_desc_scales(xs + 512 * h));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (64 * j < left) {
#pragma unroll
                            for (int m = 0; m < MATS; ++m)
                                umma_mxf4<1>(tmem_base + m * p.n_cols, smem_desc_sw128(st + m * kMxTileBytes + 32 * j), smem_desc_sw128(xs + kMxSfBytes + 32 * j),
                                             j & 1 ? id2 : id0, sf + 8 * m + 4 * (j >> 1), sf + 8 * MATS + 4 * (j >> 1), (kt | j) != 0);
                        }
                    umma_commit(smem_u32(&bar_empty[slot]));
                    if (kt + 1 == n_kt) umma_commit(smem_u32(&bar_accum));
                }
                __syncwarp();
                if (++slot == stages) slot = 0;
            }
        }
    } else {
        Item it;
        it.rows = 0;
        if constexpr (!kIsImage<XT>) {
            // Dense activations: one item, at most kMxDenseRows rows.
            if (item0 < n_items) item_of(item0, it);
            if (it.rows > 0 && n_kt > 0) {
                // lane r: the row of X of activation row r
                int my_src = lane;
                if (p.tiles) {
                    my_src = lane && lane < it.rows ? (int)ld_l2_u32(p.order + it.first + lane) : it.pair0;  // (a tile of one pair, as most are: no load)
                    if (p.pairs_per_row > 1) my_src /= p.pairs_per_row;
                }
                // A warp quantises 256 columns of a row at a time, lane 4 b + s elements 8 s .. 8 s + 7 of block b, with the next row's loads under way.
                // Up to eight column tiles the warps stand on one each, several rows abreast.
                const int b = lane >> 2, s = lane & 3, w = warp - 2;
                const int abreast = n_kt < kMxQuantWarps ? kMxQuantWarps / n_kt : 1, r0 = w / n_kt;
                if (r0 < abreast) {
                    for (int kt = w - r0 * n_kt; kt < n_kt; kt += kMxQuantWarps) {
                        const int k = (kt0 + kt) * kMxTileK + 8 * lane;
                        const XT* x = static_cast<const XT*>(p.X) + k;
                        const uint32_t at = x_base + (uint32_t)kt * x_step, to = at + kMxSfBytes + 4 * s, sc_to = at + (uint32_t)((lane >> 4) * 512);
                        MxEight<XT> v, next;
                        v.clear();
                        next.clear();
                        int64_t src = __shfl_sync(0xffffffffu, my_src, r0 & 31);
                        if (r0 < it.rows && k < p.K) v.load(x + src * p.K);
                        for (int r = r0; r < it.rows; r += abreast) {
                            src = __shfl_sync(0xffffffffu, my_src, (r + abreast) & 31);
                            if (r + abreast < it.rows && k < p.K) next.load(x + src * p.K);
                            uint32_t sc;
                            const uint32_t q = mx_quantise8(v, sc);
                            uint32_t word = sc << (8 * (b & 3));
                            word |= __shfl_xor_sync(0xffffffffu, word, 4);
                            word |= __shfl_xor_sync(0xffffffffu, word, 8);
                            sts32(to + (uint32_t)(r >> 3) * 1024u + (uint32_t)(r & 7) * 128u + ((uint32_t)(b ^ (r & 7)) << 4), q);
                            if ((lane & 15) == 0) sts32(sc_to + (uint32_t)r * 16u, word);
                            v = next;
                        }
                    }
                }
                fence_proxy_async_smem();  // generic-proxy writes -> visible to the tensor cores
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bar_x));
            }
        }
        const int r = (warp & 3) * 32 + lane;  // weight row of the tile = TMEM lane
        const uint32_t tlane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        if (warp >= 6) {
            // (quantisation only)
            if (p.split_log2) mx_cluster_wait();
        } else if (p.split_log2 == 0) {
            uint32_t phase = 0;
            bool ok = true;
            for (int i = item0; ok && i < n_items; i += item_step) {
                item_of(i, it);
                const int64_t n = (int64_t)it.row_tile * kMxTileRows + r;
                const float bv = p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, (size_t)it.expert * p.N + n) : 0.f;
                // lane x: the pair of activation row c + x of the 32 columns at hand
                int my_pair = p.tiles && lane < it.rows ? (int)ld_l2_u32(p.order + it.first + lane) : 0;
                if (!(ok = mx_warp_wait(smem_u32(&bar_accum), phase, &abort_flag, p.status, kDevTimeoutMma))) break;
                phase ^= 1;
                tc_fence_after();
                for (int c = 0; c < it.rows; c += 16) {
                    if (c && (c & 31) == 0) my_pair = p.tiles && c + lane < it.rows ? (int)ld_l2_u32(p.order + it.first + c + lane) : 0;
                    uint32_t a[MATS][16];
#pragma unroll
                    for (int m = 0; m < MATS; ++m) tmem_ld16(tlane + (uint32_t)(m * p.n_cols + c), a[m]);
                    tmem_ld_wait();
                    if (c + 16 >= it.rows) {  // the accumulator is taken: the next item's MMAs may start
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&bar_free));
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (c + j < it.rows) {
                            const size_t row = (size_t)(p.tiles ? __shfl_sync(0xffffffffu, my_pair, (c + j) & 31) : it.first + c + j);
                            float v = __uint_as_float(a[0][j]) + bv;
                            if (MATS == 2) v = silu_times(__uint_as_float(a[0][j]), __uint_as_float(a[MATS - 1][j]));
                            if (n < p.N) store_y(p.Y, p.y_dtype, row * p.N + n, v);
                        }
                    }
                }
            }
        } else {
            // One item. Rank q adds up weight rows [q * mine, + mine) of the tile. Every rank sends it its sums of these - parts[rank][matrix][activation
            // row][mine], weight row r being row r % mine of rank r / mine - and its barrier counts the bytes.
            if (item0 < n_items) item_of(item0, it);
            const int rows = it.rows, w = warp - 2;
            if (tid == 64 && rows > 0) mbar_arrive_expect_tx(smem_u32(&bar_parts), (uint32_t)(MATS * rows) << 9);
            if (w * 32 + lane < rows) row_of[w * 32 + lane] = !p.tiles ? it.first + w * 32 + lane : w + lane ? (int)ld_l2_u32(p.order + it.first + w * 32 + lane) : it.pair0;
            asm volatile("bar.sync 1, 128;" ::: "memory");  // row_of is complete
            const uint32_t to_rank = (uint32_t)(r >> mine_log2);
            const uint32_t to = mx_map_to_rank(parts + (uint32_t)((((((int)crank * MATS * rows) << mine_log2)) + (r & (mine - 1))) * 4), to_rank);
            const uint32_t to_bar = mx_map_to_rank(smem_u32(&bar_parts), to_rank);
            const int t0 = (tid - 64) >> mine_log2;  // this thread's results: activation rows t0, t0 + split, .. of weight row x
            const int x = (tid - 64) & (mine - 1);
            const int64_t n = (int64_t)it.row_tile * kMxTileRows + (int)crank * mine + x;
            const float bv = rows > 0 && p.bias && n < p.N ? load_bias(p.bias, p.bias_dtype, (size_t)it.expert * p.N + n) : 0.f;
            bool live = true;
            mx_cluster_wait();
            if (rows > 0 && n_kt > 0) live = mx_warp_wait(smem_u32(&bar_accum), 0, &abort_flag, p.status, kDevTimeoutMma);
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
            // (a peer that waits in vain for something gives up before this does)
            const bool ok = rows > 0 && mx_warp_wait<kMbarCluster>(smem_u32(&bar_parts), 0, &abort_flag, p.status, kDevTimeoutPeer, 4 * kWaitLimitNs);
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
                    store_y(p.Y, p.y_dtype, (size_t)row_of[t] * p.N + n, v);
                }
            }
        }
    }
    __syncwarp();
    if (p.split_log2 && warp < 2) mx_cluster_wait();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) {  // given up: let the copies in flight land before the CTA's shared memory is given away
        for (int s = 0; s < p.n_stages; ++s)
            if (used >> s & 1u) mbar_wait_bounded(smem_u32(&bar_full[s]), parity >> s & 1u, p.status, kDevTimeoutFull, 1u << 12);
    }
    if (warp == 1) {
        __syncwarp();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

constexpr int mx_budget(int per_sm) { return (per_sm == 3 ? 74 : per_sm == 2 ? 111 : 222) * 1024; }

// CTAs that are resident at a time in clusters of 2^log2 where an SM has room for one: a cluster lies within one group of SMs, which the larger ones do not fill
// (of 148 SMs clusters of 2 / 4 / 8 take 148 / 132 / 120). One cluster too many is a second wave: 72 rows of 2048 x 8192 in 16 clusters of 8 took 15.5 us, in 16 of 4
// 11.9; of 4608 x 6144 in 36 of 4 21.0, of 2 16.2. Asked only there. With two CTAs an SM clusters of eight hold about 264, which 34 to 37 row tiles pass (4608 x 4096
// at 17 / 32 / 48 rows 9.8 / 10.8 / 12.5 us, 4096 x 4096 7.2 / 7.8 / 8.7); dense rows were the faster for the largest split all the same (6400 x 8192, one row: 9.2 us for 10.7).
static int64_t mx_resident(int log2, int sms) {
    static std::atomic<int> known[64][4] = {};
    int dev = 0, n = 0;
    if (log2 == 0 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sms;
    if ((n = known[dev][log2].load(std::memory_order_relaxed)) != 0) return n;
    auto kern = mx4_gemm_kernel<1, void>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << log2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << log2);
    cfg.blockDim = dim3(kMxThreads<void>);
    cfg.dynamicSmemBytes = mx_budget(1);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return sms;
    }
    known[dev][log2].store(n << log2, std::memory_order_relaxed);
    return n << log2;
}

template <int MATS, typename XT>
static int launch_mx_gemm(const MxParams& q, int64_t x_tiles, int64_t rows_most, int sms, cudaStream_t st) {
    auto kern = mx4_gemm_kernel<MATS, XT>;
    MxParams p = q;
    const int per_sm = kIsImage<XT> || MATS == 2 ? 2 : 3;
    const int64_t row_tiles = mx_row_tiles(p.N), tiles = x_tiles * row_tiles;
    if (tiles > (1LL << 30)) return fail(B200Q_ERR_UNSUPPORTED, "mx4: %lld x %lld tiles are more than one launch takes", (long long)x_tiles, (long long)row_tiles);
    p.x_tiles = (int)x_tiles;
    p.row_tiles = (int)row_tiles;
    // CTAs to fill the SMs: two of an image's, and of gated dense ones (111 KB each), three of the others (74 KB). K is split while they are fewer and
    // every share keeps two column tiles or more.
    p.split_log2 = 0;
    while (p.split_log2 < 3 && tiles << (p.split_log2 + 1) <= (int64_t)per_sm * sms && p.k_tiles >= 4 << p.split_log2) ++p.split_log2;
    if (!kIsImage<XT>)  // every share's activations have to fit beside three stages
        while ((p.k_tiles + (1 << p.split_log2) - 1) >> p.split_log2 > kMxDenseTiles) ++p.split_log2;
    p.n_cols = rows_most >= kMxTileRows ? kMxTileRows : (int)((rows_most + 15) & ~15);
    int split, fixed, budget;
    for (;; --p.split_log2) {
        split = 1 << p.split_log2;
        p.split_tiles = (p.k_tiles + split - 1) / split;
        // (the groups of a product that comes here have a dozen rows on average: stages for 128 would be half empty)
        p.few_rows = p.tiles && split == 1 && p.n_cols > 32 ? 32 : p.n_cols;
        const int x_step = p.few_rows * 128 + kMxSfBytes;
        p.stage_bytes = MATS * kMxTileBytes + (kIsImage<XT> ? x_step : 0);
        p.big_bytes = MATS * kMxTileBytes + kMxSfBytes + p.n_cols * 128;
        fixed = (kIsImage<XT> ? 0 : p.split_tiles * x_step) + (split > 1 ? MATS * p.n_cols * 512 : 0);  // activations, parts
        // Shared memory of an SM's `per_sm` CTAs; of fewer where three stages would not fit. The stages' scales take TMEM columns behind the accumulators.
        budget = mx_budget(per_sm);
        if (fixed + 3 * p.stage_bytes > budget) budget = mx_budget(2);
        if (fixed + 3 * p.stage_bytes > budget || MATS * p.n_cols + 24 * (MATS + 1) > 256) budget = mx_budget(1);
        // a split whose parts leave an SM room for one CTA only goes as far as those are resident
        if (!kIsImage<XT> || split == 1 || budget < mx_budget(1) || tiles * split <= mx_resident(p.split_log2, sms)) break;
    }
    const int acc = MATS * p.n_cols, sf = 8 * (MATS + 1);
    p.n_stages = (budget - fixed) / p.stage_bytes;
    if (p.n_stages > kMxMaxStages) p.n_stages = kMxMaxStages;
    if (!kIsImage<XT> && p.n_stages > p.split_tiles) p.n_stages = p.split_tiles;
    const int most = budget == mx_budget(1) ? 512 : 256;
    while (acc + p.n_stages * sf > most) --p.n_stages;
    // At least one of either kind. Three or more of the first, but for gated groups of more than 80 rows with K split, whose parts take 96 KB or more: two, from 113 rows on one
    // (20 tokens, 7 of 16 experts, gated 496 x 3200: 17.1 us; in the wide form 12.9).
    p.big_stages = p.n_stages * p.stage_bytes / p.big_bytes;
    p.tmem_cols = 32u;
    while ((int)p.tmem_cols < acc + p.n_stages * sf) p.tmem_cols *= 2;
    const size_t smem = mx_smem_for_tmem((size_t)p.n_stages * p.stage_bytes + fixed + 1024, p.tmem_cols, split > 1);
    static bool configured[64] = {};
    int dev = 0;
    B200Q_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        B200Q_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    // an image's products: persistent CTAs, whose ring runs on from item to item
    int64_t ctas = tiles * split;
    const int64_t resident = (int64_t)sms * (budget == mx_budget(1) ? 1 : per_sm);
    if (kIsImage<XT> && split == 1 && ctas > resident) ctas = resident;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kMxThreads<XT>);
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
    B200Q_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return B200Q_OK;
}

static MxParams mx_params(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, const int* plan,
                          int64_t pairs, int E, int* status, int64_t* x_tiles) {
    MxParams p = {};
    p.W = static_cast<const uint8_t*>(W);
    p.W_up = static_cast<const uint8_t*>(W_up);
    p.X = X;
    p.bias = bias;
    p.bias_dtype = bias_dtype;
    p.Y = Y;
    p.y_dtype = y_dtype;
    p.status = status;
    p.M = M;
    p.N = N;
    p.K = K;
    p.k_tiles = mx_k_tiles(K);
    p.pairs_per_row = 1;
    p.experts = 1;
    *x_tiles = mx_row_tiles(M);
    if (plan) {
        const MoePlanLayout l = moe_plan_layout(pairs, E);
        p.w_expert_bytes = mx_image_bytes(N, K);
        p.tiles = reinterpret_cast<const int4*>(plan + l.tiles);
        p.n_tiles = plan + l.n_tiles;
        p.order = plan + l.order;
        p.experts = E;
        *x_tiles = l.max_tiles;
    }
    return p;
}

static int g_mx4_wide = 1, g_mx4_few = kMxDenseRows;
void mx4_set_wide(int v) { g_mx4_wide = v; }
int mx4_get_wide() { return g_mx4_wide; }
void mx4_set_few(int v) { g_mx4_few = v; }
int mx4_get_few() { return g_mx4_few; }

int launch_mx4_wide(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                    int E, int early, int sms, int* status, cudaStream_t st);

// X an image: M rows of one matrix (plan == nullptr), or the experts of a plan (buffer laid out for `pairs` pairs and E experts). `early`: the launch
// before this one in the stream is the quantisation that made X.
int launch_mx4_gemm(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                    int E, int early, int sms, int* status, cudaStream_t st) {
    // Where the wide tiles are the faster ones, by measurement (small tiles' time grows with the rows, the wide ones' hardly; us, small and wide):
    // row tiles for every SM, nothing to split: 14336 x 4096 at 32 / 48 / 64 rows 12.7 13.4 / 14.9 13.6 / 16.9 13.6;
    // too many for a split by four with one CTA an SM, as it is from 65 rows: 8192 x 8192 at 64 / 72 / 87 15.2 16.8 / 18.6 17.0 / 20.3 17.0, 4608 x 4096 at 48 / 72 / 87
    // 12.3 11.7 / 15.1 11.8 / 16.8 11.8;
    // fewer: 4096 x 4096 at 64 / 80 / 88 / 128 9.6 11.5 / 11.8 11.8 / 12.7 12.0 / 15.4 12.2, 1024 x 4096 7.1 10.9 / 8.2 10.9 / 9.0 11.5 / 11.0 11.8;
    // and with many columns, which the wide form does not split: 2560 x 6912 at 80 / 96 / 112 / 128 12.4 14.6 / 13.3 14.7 / 14.6 14.8 / 16.0 15.0, 4096 x 14336 15.6 23.0 /
    // 16.8 23.1 / 18.0 23.2 / 19.9 23.9, 512 x 7168 8.4 13.9 / 9.1 14.1 / 10.5 15.1 / 11.3 15.1, and at 200 / 300 rows 11.5 15.3 / 12.0 15.4.
    // The last two lines go by rows and columns alone, set for 4096 x 4096 and 2560 x 6912: where few tiles or very long columns are left, the small tiles would still be the
    // faster ones beyond them.
    // Experts, on average 8 / 12 / 16 pairs each: 128 gated 768 x 2048 40.5 41.8 / 51.5 42.1 / 48.7 42.9, 32 of 2048 x 2048 16.4 19.7 / - / 24.8 19.6,
    // 8 gated 4096 x 4096 27.0 31.6 / - / 32.6 31.7.
    const int64_t row_tiles = mx_row_tiles(N);
    const bool many = plan ? pairs >= 12LL * E : M >= (row_tiles * 2 > sms ? 48 : row_tiles * 4 > mx_resident(2, sms) ? 65 : mx_k_tiles(K) >= 24 ? 120 : 88);
    if (g_mx4_wide == 2 || (g_mx4_wide == 1 && many))
        return launch_mx4_wide(W, W_up, X, bias, bias_dtype, Y, y_dtype, M, N, K, plan, pairs, E, early, sms, status, st);
    int64_t x_tiles;
    MxParams p = mx_params(W, W_up, X, bias, bias_dtype, Y, y_dtype, M, N, K, plan, pairs, E, status, &x_tiles);
    p.early = early && pdl_option() >= 0;
    const int64_t rows_most = plan ? pairs : M;
    return W_up ? launch_mx_gemm<2, void>(p, x_tiles, rows_most, sms, st) : launch_mx_gemm<1, void>(p, x_tiles, rows_most, sms, st);
}

// Whether a product of so many rows (of one matrix, or pairs of a plan: no group can be larger) runs as one launch on dense X.
bool mx4_dense_takes(int64_t rows, int K) {
    return rows <= (g_mx4_few < kMxDenseRows ? g_mx4_few : kMxDenseRows) && mx_k_tiles(K) <= 8 * kMxDenseTiles;
}

// X dense, of x_dtype (which the bias has too), for a product that mx4_dense_takes.
int launch_mx4_dense(const void* W, const void* W_up, const void* X, int x_dtype, const void* bias, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                     int pairs_per_row, int E, int sms, int* status, cudaStream_t st) {
    int64_t x_tiles;
    MxParams p = mx_params(W, W_up, X, bias, x_dtype, Y, y_dtype, M, N, K, plan, pairs, E, status, &x_tiles);
    p.pairs_per_row = pairs_per_row;
    auto run = [&](auto zero) {
        using XT = decltype(zero);
        return W_up ? launch_mx_gemm<2, XT>(p, x_tiles, kMxDenseRows, sms, st) : launch_mx_gemm<1, XT>(p, x_tiles, kMxDenseRows, sms, st);
    };
    return x_dtype == B200Q_DT_F32 ? run(0.f) : x_dtype == B200Q_DT_F16 ? run(__half()) : run(__nv_bfloat16());
}

}  // namespace b200q
