// The routing of a sparse expert layer: the k best experts of each token with their weights, the grouping of the token-expert
// pairs by expert, and the weighted sum of the experts' results.
//
// Selection compares the logits themselves (as integers that order like them), so that it does not depend on how the softmax rounds;
// ties go to the lower expert. Weights are FP32 softmax values. The grouping is a stable counting sort: no atomics, the same order on
// every run. All of it is bound by launches and latency at the sizes of a decode step; the sum is bound by memory.
#include "mx4_common.cuh"

namespace b200q {

constexpr int kRouteWarps = 8;
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

// One warp, one token: lane l holds experts l, l + 32, ...
template <typename T, int PER_LANE>
__device__ __forceinline__ void route_token(const T* logits, int E, int k, bool normalize, float scale, int* ids, float* weights, int lane) {
    uint32_t key[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int e = lane + 32 * i;
        key[i] = 0u;
        if (e < E) {
            float v;
            if constexpr (sizeof(T) == 4) v = __uint_as_float(ld_dep_u32(logits + e));
            else {
                const unsigned short h = (unsigned short)ld_dep_u16(logits + e);
                v = to_f32<T>(*reinterpret_cast<const T*>(&h));
            }
            key[i] = route_key(v);
        }
    }
    uint32_t best = 0u;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) best = max(best, key[i]);
    const uint32_t top_key = __reduce_max_sync(0xffffffffu, best);
    const float top = route_value(top_key);
    float sum = 0.f;
    if (!normalize) {
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (key[i]) sum += route_exp(route_value(key[i]), top);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    int my_id = -1;  // lane j keeps the j-th choice
    float my_e = 0.f;
    for (int j = 0; j < k; ++j) {
        uint32_t b = 0u;
        int at = kMaxExperts;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (key[i] > b) { b = key[i]; at = lane + 32 * i; }
        const uint32_t m = __reduce_max_sync(0xffffffffu, b);
        if (m == 0u) break;  // no expert left
        const int e = __reduce_min_sync(0xffffffffu, b == m ? at : kMaxExperts);
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (lane + 32 * i == e) key[i] = 0u;
        const float w = route_exp(route_value(m), top);
        if (normalize) sum += w;
        if (lane == j) { my_id = e; my_e = w; }
    }
    if (lane < k) {
        ids[lane] = my_id;
        weights[lane] = my_id < 0 ? 0.f : my_e / sum * scale;
    }
}

template <typename T, int PER_LANE>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_topk_kernel(const T* logits, int64_t tokens, int E, int k, int normalize, float scale, int* ids, float* weights) {
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31;
    for (int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < tokens; t += (int64_t)gridDim.x * kRouteWarps)
        route_token<T, PER_LANE>(logits + t * E, E, k, normalize != 0, scale, ids + t * k, weights + t * k, lane);
}

// ---- grouping: counting sort in three passes over blocks of 1024 pairs -------------------------------------------------
// pass 1: hist[block][e] = pairs of the block that go to expert e
__global__ void __launch_bounds__(kPlanBlockPairs) moe_count_kernel(const int* ids, int64_t pairs, int E, int* hist) {
    extern __shared__ int count[];
    grid_dep_launch();
    grid_dep_wait();
    for (int e = threadIdx.x; e < E; e += kPlanBlockPairs) count[e] = 0;
    __syncthreads();
    const int64_t s = (int64_t)blockIdx.x * kPlanBlockPairs + threadIdx.x;
    if (s < pairs) {
        const int e = (int)ld_dep_u32(ids + s);
        if ((unsigned)e < (unsigned)E) atomicAdd(&count[e], 1);  // (counts do not depend on the order)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kPlanBlockPairs) hist[(int64_t)blockIdx.x * E + e] = count[e];
}

// pass 2, one block, thread e is expert e: hist becomes the first place of each block's pairs; offsets and tiles
__global__ void __launch_bounds__(kMaxExperts) moe_scan_kernel(int E, int blocks, int* hist, int* offsets, int* n_tiles, int4* tiles, int4* units) {
    __shared__ int warp_pairs[32], warp_tiles[32], warp_units[32];
    grid_dep_launch();
    grid_dep_wait();
    const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
    int total = 0;
    if (e < E)
        for (int b = 0; b < blocks; ++b) total += (int)ld_dep_u32(hist + (int64_t)b * E + e);
    const int my_tiles = (total + kMxTileRows - 1) / kMxTileRows, my_units = (my_tiles + 1) / 2;
    int pairs_to = total, tiles_to = my_tiles, units_to = my_units;  // inclusive sums
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, pairs_to, o), c = __shfl_up_sync(0xffffffffu, tiles_to, o), d = __shfl_up_sync(0xffffffffu, units_to, o);
        if (lane >= o) { pairs_to += a; tiles_to += c; units_to += d; }
    }
    if (lane == 31) { warp_pairs[warp] = pairs_to; warp_tiles[warp] = tiles_to; warp_units[warp] = units_to; }
    __syncthreads();
    for (int w = 0; w < warp; ++w) { pairs_to += warp_pairs[w]; tiles_to += warp_tiles[w]; units_to += warp_units[w]; }
    if (e < E) {
        int at = pairs_to - total;
        offsets[e] = at;
        for (int i = 0; i < my_tiles; ++i) tiles[tiles_to - my_tiles + i] = make_int4(e, at + i * kMxTileRows, min(kMxTileRows, total - i * kMxTileRows), 0);
        for (int i = 0; i < my_units; ++i)
            units[units_to - my_units + i] = make_int4(e, at + i * 2 * kMxTileRows, min(2 * kMxTileRows, total - i * 2 * kMxTileRows), tiles_to - my_tiles + 2 * i);
        for (int b = 0; b < blocks; ++b) {
            int* h = hist + (int64_t)b * E + e;
            const int c = (int)ld_dep_u32(h);
            *h = at;
            at += c;
        }
    }
    if (e == kMaxExperts - 1) {
        offsets[E] = pairs_to;
        n_tiles[0] = tiles_to;
        n_tiles[1] = units_to;
    }
}

// pass 3: each pair to its place, stable
__global__ void __launch_bounds__(kPlanBlockPairs) moe_place_kernel(const int* ids, int64_t pairs, int E, const int* hist, const int* offsets, const int* n_tiles,
                                                                    const int4* tiles, int* order, int* place) {
    extern __shared__ unsigned short before[];  // [32 warps][E]: pairs of earlier warps of this block
    grid_dep_launch();
    grid_dep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < 32 * E; i += kPlanBlockPairs) before[i] = 0;
    __syncthreads();
    const int64_t s = (int64_t)blockIdx.x * kPlanBlockPairs + threadIdx.x;
    int e = -1;
    if (s < pairs) e = (int)ld_dep_u32(ids + s);
    if ((unsigned)e >= (unsigned)E) e = -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && rank == 0) before[warp * E + e] = (unsigned short)__popc(same);
    __syncthreads();
    for (int x = threadIdx.x; x < E; x += kPlanBlockPairs) {
        int sum = 0;
        for (int w = 0; w < 32; ++w) {
            const int c = before[w * E + x];
            before[w * E + x] = (unsigned short)sum;
            sum += c;
        }
    }
    __syncthreads();
    if (s < pairs) {
        if (e >= 0) {
            const int at = (int)ld_dep_u32(hist + (int64_t)blockIdx.x * E + e) + before[warp * E + e] + rank;
            order[at] = (int)s;
            // the expert's first tile: tiles of one expert are neighbours, found by bisection on their first places
            int lo = 0, hi = (int)ld_dep_u32(n_tiles) - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((int)ld_dep_u32(&tiles[mid].y) <= at) lo = mid;
                else hi = mid - 1;
            }
            place[s] = lo * kMxTileRows + at - (int)ld_dep_u32(&tiles[lo].y);
        } else {
            place[s] = -1;
        }
        if (s >= (int64_t)(int)ld_dep_u32(offsets + E)) order[s] = -1;  // behind the last pair that has an expert
    }
}

// ---- out[t] = sum_j weights[t][j] * y[t][j], j in order, FP32; pairs without an expert are not read -----------------------
template <typename T, int VEC>
__global__ void __launch_bounds__(256) moe_combine_kernel(const T* y, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, T* out) {
    grid_dep_launch();
    grid_dep_wait();
    const int per_row = (N + VEC - 1) / VEC;
    const int64_t items = tokens * per_row, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < items; i += step) {
        const int64_t t = i / per_row;
        const int n = (int)(i - t * per_row) * VEC;
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
        for (int j = 0; j < k; ++j) {
            const int e = (int)ld_dep_u32(ids + t * k + j);
            if ((unsigned)e >= (unsigned)E) continue;
            const float w = __uint_as_float(ld_dep_u32(weights + t * k + j));
            const T* src = y + (t * k + j) * N + n;
            if constexpr (VEC == 1) {
                acc[0] = fmaf(w, to_f32<T>(*src), acc[0]);
            } else {
                union {
                    uint4 q;
                    T e[VEC];
                } u;
                u.q = ld_dep_u4(src);
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w, to_f32<T>(u.e[v]), acc[v]);
            }
        }
        if constexpr (VEC == 1) {
            out[t * N + n] = from_f32<T>(acc[0]);
        } else {
            union {
                uint4 q;
                T e[VEC];
            } u;
#pragma unroll
            for (int v = 0; v < VEC; ++v) u.e[v] = from_f32<T>(acc[v]);
            *reinterpret_cast<uint4*>(out + t * N + n) = u.q;
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
template <typename T>
static cudaError_t topk_typed(const void* logits, int64_t tokens, int E, int k, int normalize, float scale, int* ids, float* weights, int sms, cudaStream_t st) {
    int64_t blocks = (tokens + kRouteWarps - 1) / kRouteWarps;
    if (blocks > (int64_t)sms * 8) blocks = (int64_t)sms * 8;
    const T* l = static_cast<const T*>(logits);
    const bool dep = pdl_option() >= 0;
    const dim3 grid((unsigned)blocks), block(kRouteWarps * 32);
    if (E <= 64) return launch_dep(dep, moe_topk_kernel<T, 2>, grid, block, 0, st, l, tokens, E, k, normalize, scale, ids, weights);
    if (E <= 256) return launch_dep(dep, moe_topk_kernel<T, 8>, grid, block, 0, st, l, tokens, E, k, normalize, scale, ids, weights);
    return launch_dep(dep, moe_topk_kernel<T, kRouteValues>, grid, block, 0, st, l, tokens, E, k, normalize, scale, ids, weights);
}

int launch_moe_topk(const void* logits, int dtype, int64_t tokens, int E, int k, int normalize, float scale, int* ids, float* weights, int sms, cudaStream_t st) {
    if (dtype == B200Q_DT_F32) B200Q_CUDA_TRY(topk_typed<float>(logits, tokens, E, k, normalize, scale, ids, weights, sms, st));
    else if (dtype == B200Q_DT_F16) B200Q_CUDA_TRY(topk_typed<__half>(logits, tokens, E, k, normalize, scale, ids, weights, sms, st));
    else B200Q_CUDA_TRY(topk_typed<__nv_bfloat16>(logits, tokens, E, k, normalize, scale, ids, weights, sms, st));
    return B200Q_OK;
}

int launch_moe_plan(const int* ids, int64_t pairs, int E, int* plan, cudaStream_t st) {
    const MoePlanLayout l = moe_plan_layout(pairs, E);
    int *offsets = plan, *order = plan + l.order, *place = plan + l.place, *n_tiles = plan + l.n_tiles, *hist = plan + l.hist;
    int4 *tiles = reinterpret_cast<int4*>(plan + l.tiles), *units = reinterpret_cast<int4*>(plan + l.units);
    const bool dep = pdl_option() >= 0;
    const dim3 grid((unsigned)l.hist_blocks), block(kPlanBlockPairs);
    if (l.hist_blocks) B200Q_CUDA_TRY(launch_dep(dep, moe_count_kernel, grid, block, (size_t)E * 4, st, ids, pairs, E, hist));
    B200Q_CUDA_TRY(launch_dep(dep, moe_scan_kernel, dim3(1), dim3(kMaxExperts), 0, st, E, l.hist_blocks, hist, offsets, n_tiles, tiles, units));
    if (l.hist_blocks) {
        const size_t smem = (size_t)64 * E;
        static bool configured[64] = {};
        int dev = 0;
        B200Q_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            B200Q_CUDA_TRY(cudaFuncSetAttribute(moe_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * kMaxExperts));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        B200Q_CUDA_TRY(launch_dep(dep, moe_place_kernel, grid, block, smem, st, ids, pairs, E, static_cast<const int*>(hist), static_cast<const int*>(offsets),
                                  static_cast<const int*>(n_tiles), static_cast<const int4*>(tiles), order, place));
    }
    return B200Q_OK;
}

template <typename T>
static cudaError_t combine_typed(const void* y, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, void* out, int sms, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool dep = pdl_option() >= 0;
    const bool wide = N % V == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    int64_t blocks = (tokens * (wide ? N / V : N) + 255) / 256;
    if (blocks > (int64_t)sms * 16) blocks = (int64_t)sms * 16;
    const dim3 grid((unsigned)blocks), block(256);
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
