// The routing of a sparse expert layer: the k best experts of each token with their weights, the grouping of the token-expert
// pairs by expert, and the weighted sum of the experts' results.
//
// Selection compares the logits themselves (as integers that order like them), so that it does not depend on how the softmax rounds;
// ties go to the lower expert. Weights are FP32 softmax values. The grouping is a stable counting sort: no atomics, the same order on
// every run. All of it is bound by launches and latency at the sizes of a decode step; the sum is bound by memory.
#include <type_traits>

#include "mx4_common.cuh"

namespace b200q {

constexpr int kRouteValues = kMaxExperts / 32;

// Unsigned integers that order like the floats, NaN and -inf as 0 (never chosen).
__device__ __forceinline__ uint32_t route_key(float v) {
    if (!(v > __uint_as_float(0xFF800000u))) return 0u;
    const uint32_t u = __float_as_uint(v + 0.f);  // (-0 and 0 are a tie)
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

// exp(v - top), where an infinite top takes all
__device__ __forceinline__ float route_exp(float v, float top) {
    if (top == __uint_as_float(0x7F800000u)) return v == top ? 1.f : 0.f;
    return expf(v - top);
}

// One warp, TOKENS neighbouring tokens of which `have` exist: lane l holds experts l, l + 32, ... of each. A choice is a chain of a scan and two
// warp reductions; the tokens' chains run side by side. `keep`, where not nullptr, gets the ids too.
template <typename T, int PER_LANE, int TOKENS>
__device__ __forceinline__ void route_tokens(const T* logits, int have, int E, int k, bool normalize, float scale, int* ids, float* weights, int* keep, int lane) {
    uint32_t key[TOKENS][PER_LANE];
#pragma unroll
    for (int u = 0; u < TOKENS; ++u)
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int e = lane + 32 * i;
            key[u][i] = 0u;
            if (u < have && e < E) {
                float v;
                if constexpr (sizeof(T) == 4) v = __uint_as_float(ld_dep_u32(logits + (int64_t)u * E + e));
                else {
                    const unsigned short h = (unsigned short)ld_dep_u16(logits + (int64_t)u * E + e);
                    v = to_f32<T>(*reinterpret_cast<const T*>(&h));
                }
                key[u][i] = route_key(v);
            }
        }
    float top[TOKENS], sum[TOKENS], my_e[TOKENS];
    int my_id[TOKENS];  // lane j keeps the j-th choice
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) {
        uint32_t best = 0u;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) best = max(best, key[u][i]);
        top[u] = route_value(__reduce_max_sync(0xffffffffu, best));
        sum[u] = my_e[u] = 0.f;
        my_id[u] = -1;
    }
    if (!normalize) {
#pragma unroll
        for (int u = 0; u < TOKENS; ++u) {
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (key[u][i]) sum[u] += route_exp(route_value(key[u][i]), top[u]);
#pragma unroll
            for (int o = 16; o; o >>= 1) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
        }
    }
    for (int j = 0; j < k; ++j) {
#pragma unroll
        for (int u = 0; u < TOKENS; ++u) {
            uint32_t b = 0u;
            int at = kMaxExperts;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (key[u][i] > b) { b = key[u][i]; at = lane + 32 * i; }
            const uint32_t m = __reduce_max_sync(0xffffffffu, b);
            const int e = __reduce_min_sync(0xffffffffu, b == m && m ? at : kMaxExperts);  // kMaxExperts: no expert left
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (lane + 32 * i == e) key[u][i] = 0u;
            if (m) {
                const float w = route_exp(route_value(m), top[u]);
                if (normalize) sum[u] += w;
                if (lane == j) { my_id[u] = e; my_e[u] = w; }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < TOKENS; ++u)
        if (u < have && lane < k) {
            ids[u * k + lane] = my_id[u];
            weights[u * k + lane] = my_id[u] < 0 ? 0.f : my_e[u] / sum[u] * scale;
            if (keep) keep[u * k + lane] = my_id[u];
        }
}

// ---- routing and grouping ------------------------------------------------------------------------------------------
// The pairs are cut into at most 128 ranges of whole tokens. Pass 1 chooses the experts of a range's tokens (or reads given ids) and counts the
// range's pairs by expert; in pass 2 every block adds up the counts of the ranges before its own - 128 x E integers at most, from the L2 - and
// puts its pairs into their places, chunk by chunk, in order: a pair's rank in its chunk is the number of equal ids in the warps before and in the lanes
// before. One range (up to 1024 pairs, a decode step) does both in one launch.
struct RouteParams {
    const void* logits;   // nullptr: ids are given
    int64_t tokens, range_tokens;
    int E, k, normalize, ranges;
    float scale;
    int* ids;
    float* weights;
    // plan (see MoePlanLayout); nullptr: none is wanted
    int *offsets, *order, *place, *n_tiles, *hist;
    int4 *tiles, *units;
};

constexpr int kRouteThreads = 1024, kLeastPairs = 64;  // of a range

// The experts of tokens [t0, t1), the block's warps side by side: four tokens a warp where there are several for each
template <typename T, int PER_LANE>
__device__ __forceinline__ void route_choose(const RouteParams& p, int64_t t0, int64_t t1, int* keep) {
    constexpr int kTokens = PER_LANE <= 8 ? 4 : 1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const T* logits = static_cast<const T*>(p.logits);
    if (kTokens > 1 && t1 - t0 > warps) {
        for (int64_t t = t0 + kTokens * warp; t < t1; t += kTokens * warps)
            route_tokens<T, PER_LANE, kTokens>(logits + t * p.E, (int)min(t1 - t, (int64_t)kTokens), p.E, p.k, p.normalize != 0, p.scale, p.ids + t * p.k, p.weights + t * p.k,
                                               keep ? keep + (t - t0) * p.k : nullptr, lane);
    } else {
        for (int64_t t = t0 + warp; t < t1; t += warps)
            route_tokens<T, PER_LANE, 1>(logits + t * p.E, 1, p.E, p.k, p.normalize != 0, p.scale, p.ids + t * p.k, p.weights + t * p.k, keep ? keep + (t - t0) * p.k : nullptr, lane);
    }
}

// Pairs [s0, s1) of the calling block to their places. smem: 3 E ints, then (THREADS / 32 + 1) E shorts: pairs of each
// warp and expert, made into those of the warps before, and of the chunk.
// ONE: this is the only range; its counts are in the first E ints and its ids in `kept`.
template <int THREADS, bool ONE>
__device__ __forceinline__ void route_place(const RouteParams& p, int64_t s0, int64_t s1, int range, int* smem, const int* kept) {
    constexpr int kWarps = THREADS / 32, kMine = (kMaxExperts + THREADS - 1) / THREADS;  // a thread has up to kMine neighbouring experts
    __shared__ int sums[3][kWarps];
    int *next = smem, *first = smem + p.E, *tile0 = smem + 2 * p.E;  // next free place, first place and first tile of each expert
    unsigned short* before = reinterpret_cast<unsigned short*>(smem + 3 * p.E);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = p.E;
    // counts of all ranges and of those before this one; as many threads to an expert as there are, each with a part of the ranges
    if (ONE) {
        for (int e = tid; e < E; e += THREADS) {
            first[e] = next[e];
            next[e] = 0;
        }
    } else {
        for (int e = tid; e < E; e += THREADS) next[e] = first[e] = 0;
        __syncthreads();
        const int parts = max(THREADS / E, 1), per = (p.ranges + parts - 1) / parts;
        for (int i = tid; i < parts * E; i += THREADS) {
            const int part = i / E, e = i - part * E, r1 = min((part + 1) * per, p.ranges);
            int all = 0, earlier = 0;
#pragma unroll 8
            for (int r = part * per; r < r1; ++r) {
                const int c = (int)ld_dep_u32(p.hist + (int64_t)r * E + e);
                all += c;
                earlier += r < range ? c : 0;
            }
            if (all) atomicAdd(&first[e], all);
            if (earlier) atomicAdd(&next[e], earlier);
        }
    }
    const int chunk_warps = (int)min((s1 - s0 + 31) >> 5, (int64_t)kWarps);  // warps that have pairs
    __syncthreads();
    // running sums of pairs, tiles and units over the experts
    int pairs[kMine], sum[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int e = tid * kMine + i;
        pairs[i] = e < E ? first[e] : 0;
        const int t = (pairs[i] + kMxTileRows - 1) / kMxTileRows;
        sum[0] += pairs[i];
        sum[1] += t;
        sum[2] += (t + 1) >> 1;
    }
    int at[3];
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        int v = sum[c];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += up;
        }
        if (lane == 31) sums[c][warp] = v;
        at[c] = v - sum[c];
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w)
#pragma unroll
        for (int c = 0; c < 3; ++c) at[c] += sums[c][w];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int e = tid * kMine + i, n = pairs[i], t = (n + kMxTileRows - 1) / kMxTileRows, u = (t + 1) >> 1;
        if (e < E) {
            next[e] += at[0];
            first[e] = at[0];
            tile0[e] = at[1];
            if (range == 0) {
                p.offsets[e] = at[0];
                for (int x = 0; x < t; ++x) {  // (the fourth word comes from the block that places the tile's first pair)
                    int4* tile = p.tiles + at[1] + x;
                    tile->x = e;
                    tile->y = at[0] + x * kMxTileRows;
                    tile->z = min(kMxTileRows, n - x * kMxTileRows);
                }
                for (int x = 0; x < u; ++x) {
                    p.units[2 * (at[2] + x)] = make_int4(e, at[0] + x * 2 * kMxTileRows, min(2 * kMxTileRows, n - x * 2 * kMxTileRows), at[1] + 2 * x);
                    p.units[2 * (at[2] + x) + 1] = make_int4(at[2], u, 0, 0);
                }
            }
        }
        at[0] += n;
        at[1] += t;
        at[2] += u;
    }
    __shared__ int placed;
    if (tid == THREADS - 1) placed = at[0];
    if (range == 0 && tid == THREADS - 1) {
        p.offsets[E] = at[0];
        p.n_tiles[0] = at[1];
        p.n_tiles[1] = at[2];
    }
    for (int64_t c0 = s0; c0 < s1; c0 += THREADS) {
        for (int i = tid; i < chunk_warps * E; i += THREADS) before[i] = 0;
        __syncthreads();
        const int64_t s = c0 + tid;
        int e = s < s1 ? (ONE ? kept[s] : (int)ld_dep_u32(p.ids + s)) : -1;
        if ((unsigned)e >= (unsigned)E) e = -1;
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (e >= 0 && rank == 0) before[warp * E + e] = (unsigned short)__popc(same);
        __syncthreads();
        for (int x = tid; x < E; x += THREADS) {
            int run = 0;
#pragma unroll 4
            for (int w = 0; w < chunk_warps; ++w) {
                const int c = before[w * E + x];
                before[w * E + x] = (unsigned short)run;
                run += c;
            }
            before[kWarps * E + x] = (unsigned short)run;
            next[x] += run;  // the next chunk's places
        }
        __syncthreads();
        if (s < s1) {
            if (e >= 0) {
                const int place = next[e] - before[kWarps * E + e] + before[warp * E + e] + rank, i = place - first[e];
                p.order[place] = (int)s;
                p.place[s] = (tile0[e] + (i >> 7)) * kMxTileRows + (i & 127);
                if ((i & 127) == 0) p.tiles[tile0[e] + (i >> 7)].w = (int)s;
            } else {
                p.place[s] = -1;
            }
            if (s >= placed) p.order[s] = -1;  // behind the last pair that has an expert
        }
        __syncthreads();
    }
}

template <typename T, int PER_LANE>
__global__ void __launch_bounds__(kRouteThreads) moe_count_kernel(const RouteParams p) {
    extern __shared__ int count[];
    grid_dep_launch();
    grid_dep_wait();
    const int64_t t0 = (int64_t)blockIdx.x * p.range_tokens, t1 = min(t0 + p.range_tokens, p.tokens);
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) count[e] = 0;
    if constexpr (!std::is_same_v<T, void>) route_choose<T, PER_LANE>(p, t0, t1, nullptr);
    if (!p.offsets) return;
    __syncthreads();  // (the block's own ids are seen by all of its threads)
    for (int64_t s = t0 * p.k + threadIdx.x; s < t1 * p.k; s += blockDim.x) {
        const int e = (int)ld_dep_u32(p.ids + s);
        if ((unsigned)e < (unsigned)p.E) atomicAdd(&count[e], 1);  // (counts do not depend on the order)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) p.hist[(int64_t)blockIdx.x * p.E + e] = count[e];
}

__global__ void __launch_bounds__(kRouteThreads) moe_place_kernel(const RouteParams p) {
    extern __shared__ int smem_route[];
    grid_dep_launch();
    grid_dep_wait();
    const int64_t t0 = (int64_t)blockIdx.x * p.range_tokens, t1 = min(t0 + p.range_tokens, p.tokens);
    route_place<kRouteThreads, false>(p, t0 * p.k, t1 * p.k, (int)blockIdx.x, smem_route, nullptr);
}

// One range: both passes, at most 1024 pairs
template <typename T, int PER_LANE>
__global__ void __launch_bounds__(kRouteThreads) moe_route_one_kernel(const RouteParams p) {
    extern __shared__ int smem_route[];
    __shared__ int kept[kRouteThreads];
    int* count = smem_route;
    for (int e = threadIdx.x; e < p.E; e += kRouteThreads) count[e] = 0;
    grid_dep_launch();
    grid_dep_wait();
    const bool has = threadIdx.x < p.tokens * p.k;
    if constexpr (!std::is_same_v<T, void>) route_choose<T, PER_LANE>(p, 0, p.tokens, kept);
    else if (has) kept[threadIdx.x] = (int)ld_dep_u32(p.ids + threadIdx.x);
    __syncthreads();
    if (has && (unsigned)kept[threadIdx.x] < (unsigned)p.E) atomicAdd(&count[kept[threadIdx.x]], 1);
    __syncthreads();
    route_place<kRouteThreads, true>(p, 0, p.tokens * p.k, 0, smem_route, kept);
}

// ---- out[t] = sum_j weights[t][j] * y[t][j], j in order, FP32; pairs without an expert are not read -----------------------
// A thread has VEC neighbouring columns of a token; the loads of four pairs are in flight together.
constexpr int kCombineThreads = 256;
template <typename T, int VEC>
__global__ void __launch_bounds__(kCombineThreads) moe_combine_kernel(const T* y, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, T* out) {
    grid_dep_launch();
    grid_dep_wait();
    const int64_t n = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
    if (n >= N) return;
    constexpr int kBatch = 4;
    union Vec {
        T e[VEC];
        uint4 q;
    };
    for (int64_t t = blockIdx.y; t < tokens; t += gridDim.y) {
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
        for (int j0 = 0; j0 < k; j0 += kBatch) {
            Vec u[kBatch];
            float w[kBatch];
            bool has[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int64_t s = t * k + j0 + j;
                has[j] = j0 + j < k && ld_dep_u32(ids + s) < (uint32_t)E;
                if (has[j]) {
                    w[j] = __uint_as_float(ld_dep_u32(weights + s));
                    if constexpr (VEC == 1) u[j].e[0] = y[s * N + n];
                    else u[j].q = ld_dep_u4(y + s * N + n);
                }
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (has[j]) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w[j], to_f32<T>(u[j].e[v]), acc[v]);
                }
        }
        Vec o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) o.e[v] = from_f32<T>(acc[v]);
        if constexpr (VEC == 1) out[t * N + n] = o.e[0];
        else *reinterpret_cast<uint4*>(out + t * N + n) = o.q;
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
template <typename T, int PER_LANE>
static int route_launch(const RouteParams& q, cudaStream_t st) {
    RouteParams p = q;
    const bool dep = pdl_option() >= 0;
    const int64_t pairs = p.tokens * p.k;
    const auto smem = [&](int warps) { return (size_t)p.E * (12 + 2 * (warps + 1)) + 4; };
    const auto allow = [](auto kern) {
        static bool configured[64] = {};
        int dev = 0;
        B200Q_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            B200Q_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 80 * kMaxExperts));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        return B200Q_OK;
    };
    // One launch while a block's warps have a token each (given ids: its threads a pair): 32 tokens, 6 of 64 experts, 5.6 us in one, 33 in two 7.3. 96 tokens take
    // 10.5 in one, 7.3 in two.
    if (p.offsets && pairs <= kRouteThreads && (!p.logits || p.tokens <= kRouteThreads / 32)) {
        auto kern = moe_route_one_kernel<T, PER_LANE>;
        if (int rc = allow(kern)) return rc;
        p.ranges = 1;
        B200Q_CUDA_TRY(launch_dep(dep, kern, dim3(1), dim3(kRouteThreads), smem(kRouteThreads / 32), st, p));
        return B200Q_OK;
    }
    p.range_tokens = (p.tokens + kPlanRanges - 1) / kPlanRanges;
    const int64_t least = (kLeastPairs + p.k - 1) / p.k;
    if (p.range_tokens < least) p.range_tokens = least;
    p.ranges = (int)((p.tokens + p.range_tokens - 1) / p.range_tokens);
    // a warp for each token of a range while that makes a block (given ids: a thread for each pair)
    int64_t threads = p.logits ? p.range_tokens * 32 : (p.range_tokens * p.k + 31) & ~31;
    if (threads > kRouteThreads) threads = kRouteThreads;
    B200Q_CUDA_TRY(launch_dep(dep, moe_count_kernel<T, PER_LANE>, dim3((unsigned)p.ranges), dim3((unsigned)threads), (size_t)p.E * 4, st, p));
    if (!p.offsets) return B200Q_OK;
    if (int rc = allow(moe_place_kernel)) return rc;
    B200Q_CUDA_TRY(launch_dep(dep, moe_place_kernel, dim3((unsigned)p.ranges), dim3(kRouteThreads), smem(kRouteThreads / 32), st, p));
    return B200Q_OK;
}

static void route_plan(RouteParams& p, int* plan) {
    const MoePlanLayout l = moe_plan_layout(p.tokens * p.k, p.E);
    p.offsets = plan;
    p.order = plan + l.order;
    p.place = plan + l.place;
    p.n_tiles = plan + l.n_tiles;
    p.hist = plan + l.hist;
    p.tiles = reinterpret_cast<int4*>(plan + l.tiles);
    p.units = reinterpret_cast<int4*>(plan + l.units);
}

template <typename T>
static int route_typed(const RouteParams& p, cudaStream_t st) {
    if (p.E <= 64) return route_launch<T, 2>(p, st);
    if (p.E <= 256) return route_launch<T, 8>(p, st);
    return route_launch<T, kRouteValues>(p, st);
}

int launch_moe_route(const void* logits, int dtype, int64_t tokens, int E, int k, int normalize, float scale, int* ids, float* weights, int* plan, cudaStream_t st) {
    RouteParams p = {};
    p.logits = logits;
    p.tokens = tokens;
    p.E = E;
    p.k = k;
    p.normalize = normalize;
    p.scale = scale;
    p.ids = ids;
    p.weights = weights;
    if (plan) route_plan(p, plan);
    return dtype == B200Q_DT_F32 ? route_typed<float>(p, st) : dtype == B200Q_DT_F16 ? route_typed<__half>(p, st) : route_typed<__nv_bfloat16>(p, st);
}

int launch_moe_plan(const int* ids, int64_t tokens, int k, int E, int* plan, cudaStream_t st) {
    RouteParams p = {};
    p.tokens = tokens;
    p.E = E;
    p.k = k;
    p.ids = const_cast<int*>(ids);  // (read only: there are no logits)
    route_plan(p, plan);
    return route_launch<void, 1>(p, st);
}

template <typename T>
static cudaError_t combine_typed(const void* y, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, void* out, int sms, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool dep = pdl_option() >= 0;
    const bool wide = N % V == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int items = wide ? N / V : N;
    // few results: small blocks, so that they spread over the SMs
    const int threads = (int64_t)items * tokens >= (int64_t)sms * kCombineThreads ? kCombineThreads : 64;
    const dim3 grid(((unsigned)items + threads - 1) / threads, (unsigned)(tokens < 65535 ? tokens : 65535)), block(threads);
    if (wide) return launch_dep(dep, moe_combine_kernel<T, V>, grid, block, 0, st, static_cast<const T*>(y), ids, weights, tokens, k, N, E, static_cast<T*>(out));
    return launch_dep(dep, moe_combine_kernel<T, 1>, grid, block, 0, st, static_cast<const T*>(y), ids, weights, tokens, k, N, E, static_cast<T*>(out));
}

int launch_moe_combine(const void* y, int dtype, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, void* out, int sms, cudaStream_t st) {
    if (dtype == B200Q_DT_F32) B200Q_CUDA_TRY(combine_typed<float>(y, ids, weights, tokens, k, N, E, out, sms, st));
    else if (dtype == B200Q_DT_F16) B200Q_CUDA_TRY(combine_typed<__half>(y, ids, weights, tokens, k, N, E, out, sms, st));
    else B200Q_CUDA_TRY(combine_typed<__nv_bfloat16>(y, ids, weights, tokens, k, N, E, out, sms, st));
    return B200Q_OK;
}

}  // namespace b200q
