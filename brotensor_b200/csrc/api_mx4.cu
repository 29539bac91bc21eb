// C-ABI entry points of the MXFP4 matrices and the sparse expert layers on them (include/b200q.h): argument checks and
// launches. As in api.cu, nothing here allocates, synchronises or falls back to a CPU path.
#include "mx4_common.cuh"

namespace b200q {

int device_facts(int* sms, int** status);  // api.cu
int launch_mx4_quantise(const void* x, int x_dtype, int64_t rows, int K, void* image, const int* place, int copies, int sms, cudaStream_t st);
int launch_mx4_dequantise(const void* image, int64_t rows, int K, void* out, int out_dtype, int sms, cudaStream_t st);
int launch_mx4_pack(const void* blocks, int64_t rows, int64_t count, int K, void* image, cudaStream_t st);
int launch_mx4_gemm(const void* W, const void* W_up, const void* X, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K,
                    const int* plan, int64_t pairs, int E, int early, int sms, int* status, cudaStream_t st);
int launch_mx4_dense(const void* W, const void* W_up, const void* X, int x_dtype, const void* bias, void* Y, int y_dtype, int M, int N, int K, const int* plan, int64_t pairs,
                   int pairs_per_row, int E, int sms, int* status, cudaStream_t st);
bool mx4_dense_takes(int64_t rows, int K);
int launch_moe_route(const void* logits, int dtype, int64_t tokens, int E, int k, int normalize, float scale, int* ids, float* weights, int* plan, cudaStream_t st);
int launch_moe_plan(const int* ids, int64_t tokens, int k, int E, int* plan, cudaStream_t st);
int launch_moe_combine(const void* y, int dtype, const int* ids, const float* weights, int64_t tokens, int k, int N, int E, void* out, int sms, cudaStream_t st);

static bool dtype_ok(int dt) { return dt == B200Q_DT_F32 || dt == B200Q_DT_F16 || dt == B200Q_DT_BF16; }
static size_t dtype_size(int dt) { return dt == B200Q_DT_F32 ? 4 : 2; }
static bool on(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kMostRows = 1 << 30;  // of a dense product: row numbers stay inside 31 bits in whole pairs of tiles

static int check_k(const char* op, int K) {
    if (K <= 0 || K % 32) return fail(B200Q_ERR_BAD_ARG, "%s: K (%d) must be a positive multiple of 32", op, K);
    return B200Q_OK;
}
// Pairs of a token and an expert are numbered in 31 bits, with room for the last tile of each expert.
constexpr int64_t kMostPairs = 2147483647LL - (int64_t)kMaxExperts * kMxTileRows;
static bool experts_fit(int64_t tokens, int k, int E) {
    return tokens >= 0 && E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxExpertsPerToken && tokens <= kMostPairs / k;
}
// Sizes of a layer of experts
static int check_experts(const char* op, int64_t tokens, int k, int E) {
    if (tokens < 0) return fail(B200Q_ERR_BAD_ARG, "%s: negative token count", op);
    if (E < 1 || E > kMaxExperts) return fail(B200Q_ERR_UNSUPPORTED, "%s: E (%d) must be 1..%d", op, E, kMaxExperts);
    if (k < 1 || k > kMaxExpertsPerToken) return fail(B200Q_ERR_UNSUPPORTED, "%s: k (%d) must be 1..%d", op, k, kMaxExpertsPerToken);
    if (!experts_fit(tokens, k, E)) return fail(B200Q_ERR_UNSUPPORTED, "%s: %lld tokens of %d experts each are too many", op, (long long)tokens, k);
    return B200Q_OK;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_mx4_image_bytes(int64_t rows, int K) { return rows < 0 || K <= 0 || K % 32 ? 0 : mx_image_bytes(rows, K); }

int b200q_mx4_pack(const void* blocks, int64_t count, int64_t rows, int K, void* image, void* stream) {
    if (int rc = check_k("mx4_pack", K)) return rc;
    if (rows < 0 || count < 0) return fail(B200Q_ERR_BAD_ARG, "mx4_pack: negative shape");
    if (rows == 0 || count == 0) return B200Q_OK;
    if (!blocks || !image) return fail(B200Q_ERR_BAD_ARG, "mx4_pack: null pointer");
    if (!on(image, 16)) return fail(B200Q_ERR_BAD_ARG, "mx4_pack: the image must be 16-byte aligned");
    if (rows > 8 * 2147483647LL / count) return fail(B200Q_ERR_UNSUPPORTED, "mx4_pack: %lld x %lld rows are more than one launch takes", (long long)count, (long long)rows);
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_mx4_pack(blocks, rows, count, K, image, static_cast<cudaStream_t>(stream));
}

int b200q_mx4_quantize(const void* x, int x_dtype, int64_t rows, int K, void* image, void* stream) {
    if (!dtype_ok(x_dtype)) return fail(B200Q_ERR_BAD_ARG, "mx4_quantize: unknown dtype %d", x_dtype);
    if (int rc = check_k("mx4_quantize", K)) return rc;
    if (rows < 0) return fail(B200Q_ERR_BAD_ARG, "mx4_quantize: negative row count");
    if (rows == 0) return B200Q_OK;
    if (!x || !image) return fail(B200Q_ERR_BAD_ARG, "mx4_quantize: null pointer");
    if (!on(x, 16) || !on(image, 16)) return fail(B200Q_ERR_BAD_ARG, "mx4_quantize: x and the image must be 16-byte aligned");
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_mx4_quantise(x, x_dtype, rows, K, image, nullptr, 1, sms, static_cast<cudaStream_t>(stream));
}

int b200q_mx4_dequantize(const void* image, int64_t rows, int K, void* out, int out_dtype, void* stream) {
    if (!dtype_ok(out_dtype)) return fail(B200Q_ERR_BAD_ARG, "mx4_dequantize: unknown dtype %d", out_dtype);
    if (int rc = check_k("mx4_dequantize", K)) return rc;
    if (rows < 0) return fail(B200Q_ERR_BAD_ARG, "mx4_dequantize: negative row count");
    if (rows == 0) return B200Q_OK;
    if (!image || !out) return fail(B200Q_ERR_BAD_ARG, "mx4_dequantize: null pointer");
    if (!on(image, 16) || !on(out, 16)) return fail(B200Q_ERR_BAD_ARG, "mx4_dequantize: the image and the output must be 16-byte aligned");
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_mx4_dequantise(image, rows, K, out, out_dtype, sms, static_cast<cudaStream_t>(stream));
}

static int check_product(const char* op, const void* W, const void* X, const void* bias, int bias_dtype, const void* Y, int y_dtype) {
    if (!W || !X || !Y) return fail(B200Q_ERR_BAD_ARG, "%s: null pointer", op);
    if (!on(W, 16) || !on(X, 16)) return fail(B200Q_ERR_BAD_ARG, "%s: W and X must be 16-byte aligned", op);
    if (!on(Y, dtype_size(y_dtype))) return fail(B200Q_ERR_BAD_ARG, "%s: Y is not aligned to its element size", op);
    if (bias && !on(bias, dtype_size(bias_dtype))) return fail(B200Q_ERR_BAD_ARG, "%s: the bias is not aligned to its element size", op);
    return B200Q_OK;
}

int b200q_mx4_gemm(const void* W, const void* X_image, const void* bias, int bias_dtype, void* Y, int y_dtype, int M, int N, int K, void* stream) {
    if (!dtype_ok(y_dtype) || !dtype_ok(bias_dtype)) return fail(B200Q_ERR_BAD_ARG, "mx4_gemm: unknown dtype (y %d, bias %d)", y_dtype, bias_dtype);
    if (int rc = check_k("mx4_gemm", K)) return rc;
    if (M < 0 || N < 0) return fail(B200Q_ERR_BAD_ARG, "mx4_gemm: negative shape (M %d, N %d)", M, N);
    if (M > kMostRows) return fail(B200Q_ERR_UNSUPPORTED, "mx4_gemm: M (%d) is more than %d", M, kMostRows);
    if (M == 0 || N == 0) return B200Q_OK;
    if (int rc = check_product("mx4_gemm", W, X_image, bias, bias_dtype, Y, y_dtype)) return rc;
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_mx4_gemm(W, nullptr, X_image, bias, bias_dtype, Y, y_dtype, M, N, K, nullptr, 0, 0, 0, sms, status, static_cast<cudaStream_t>(stream));
}

size_t b200q_mx4_linear_workspace_bytes(int M, int K) { return mx4_dense_takes(M, K) ? 0 : b200q_mx4_image_bytes(M, K); }

static int check_ws(const char* op, const void* ws, size_t ws_bytes, size_t need) {
    if (need && (!ws || !on(ws, 256) || ws_bytes < need)) return fail(B200Q_ERR_WORKSPACE, "%s: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", op, need, ws ? ws_bytes : (size_t)0);
    return B200Q_OK;
}

int b200q_mx4_linear(const void* W, const void* X, int x_dtype, const void* bias, void* Y, int y_dtype, int M, int N, int K, void* ws, size_t ws_bytes,
                     void* stream) {
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return fail(B200Q_ERR_BAD_ARG, "mx4_linear: unknown dtype (x %d, y %d)", x_dtype, y_dtype);
    if (int rc = check_k("mx4_linear", K)) return rc;
    if (M < 0 || N < 0) return fail(B200Q_ERR_BAD_ARG, "mx4_linear: negative shape (M %d, N %d)", M, N);
    if (M > kMostRows) return fail(B200Q_ERR_UNSUPPORTED, "mx4_linear: M (%d) is more than %d", M, kMostRows);
    if (M == 0 || N == 0) return B200Q_OK;
    if (int rc = check_product("mx4_linear", W, X, bias, x_dtype, Y, y_dtype)) return rc;
    if (int rc = check_ws("mx4_linear", ws, ws_bytes, b200q_mx4_linear_workspace_bytes(M, K))) return rc;
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (mx4_dense_takes(M, K)) return launch_mx4_dense(W, nullptr, X, x_dtype, bias, Y, y_dtype, M, N, K, nullptr, 0, 1, 0, sms, status, st);
    if (int rc = launch_mx4_quantise(X, x_dtype, M, K, ws, nullptr, 1, sms, st)) return rc;
    return launch_mx4_gemm(W, nullptr, ws, bias, x_dtype, Y, y_dtype, M, N, K, nullptr, 0, 0, 1, sms, status, st);
}

size_t b200q_moe_plan_bytes(int64_t tokens, int k, int E) {
    if (!experts_fit(tokens, k, E)) return 0;
    return 4 * moe_plan_layout(tokens * k, E).total;
}

int b200q_moe_plan(const int32_t* ids, int64_t tokens, int k, int E, void* plan, void* stream) {
    if (int rc = check_experts("moe_plan", tokens, k, E)) return rc;
    if ((!ids && tokens) || !plan) return fail(B200Q_ERR_BAD_ARG, "moe_plan: null pointer");
    if (!on(ids, 4) || !on(plan, 16)) return fail(B200Q_ERR_BAD_ARG, "moe_plan: ids must be 4-byte and the plan 16-byte aligned");
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_moe_plan(ids, tokens, k, E, static_cast<int*>(plan), static_cast<cudaStream_t>(stream));
}

int b200q_moe_route(const void* logits, int dtype, int64_t tokens, int E, int k, int normalize, float scale, int32_t* ids, float* weights, void* plan, void* stream) {
    if (!dtype_ok(dtype)) return fail(B200Q_ERR_BAD_ARG, "moe_route: unknown dtype %d", dtype);
    if (int rc = check_experts("moe_route", tokens, k, E)) return rc;
    if (k > E) return fail(B200Q_ERR_BAD_ARG, "moe_route: k (%d) is more than E (%d)", k, E);
    if (tokens && (!logits || !ids || !weights)) return fail(B200Q_ERR_BAD_ARG, "moe_route: null pointer");
    if (!on(logits, dtype_size(dtype)) || !on(ids, 4) || !on(weights, 4) || !on(plan, 16))
        return fail(B200Q_ERR_BAD_ARG, "moe_route: logits, ids and weights must be aligned to their elements, the plan to 16 bytes");
    if (tokens == 0 && !plan) return B200Q_OK;
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_moe_route(logits, dtype, tokens, E, k, normalize, scale, ids, weights, static_cast<int*>(plan), static_cast<cudaStream_t>(stream));
}

size_t b200q_moe_mx4_workspace_bytes(int64_t tokens, int k, int E, int K) {
    if (!experts_fit(tokens, k, E) || K <= 0 || K % 32) return 0;
    return mx4_dense_takes(tokens * k, K) ? 0 : (size_t)moe_plan_layout(tokens * k, E).max_tiles * mx_k_tiles(K) * kMxTileBytes;
}

static int experts_common(const char* op, const void* W, const void* W_up, const void* X, int x_dtype, int x_per_pair, const void* plan, const void* bias, void* Y,
                          int y_dtype, int64_t tokens, int k, int E, int N, int K, void* ws, size_t ws_bytes, void* stream) {
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return fail(B200Q_ERR_BAD_ARG, "%s: unknown dtype (x %d, y %d)", op, x_dtype, y_dtype);
    if (int rc = check_k(op, K)) return rc;
    if (int rc = check_experts(op, tokens, k, E)) return rc;
    if (N < 0) return fail(B200Q_ERR_BAD_ARG, "%s: negative N (%d)", op, N);
    if (tokens == 0 || N == 0) return B200Q_OK;
    if (!plan) return fail(B200Q_ERR_BAD_ARG, "%s: null pointer", op);
    if (int rc = check_product(op, W, X, bias, x_dtype, Y, y_dtype)) return rc;
    if (!on(W_up, 16) || !on(plan, 16)) return fail(B200Q_ERR_BAD_ARG, "%s: images and the plan must be 16-byte aligned", op);
    if (int rc = check_ws(op, ws, ws_bytes, b200q_moe_mx4_workspace_bytes(tokens, k, E, K))) return rc;
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    const int64_t pairs = tokens * k;
    const int* pl = static_cast<const int*>(plan);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (mx4_dense_takes(pairs, K)) return launch_mx4_dense(W, W_up, X, x_dtype, bias, Y, y_dtype, 0, N, K, pl, pairs, x_per_pair ? 1 : k, E, sms, status, st);
    const int* place = pl + moe_plan_layout(pairs, E).place;
    if (int rc = launch_mx4_quantise(X, x_dtype, x_per_pair ? pairs : tokens, K, ws, place, x_per_pair ? 1 : k, sms, st)) return rc;
    return launch_mx4_gemm(W, W_up, ws, bias, x_dtype, Y, y_dtype, 0, N, K, pl, pairs, E, 1, sms, status, st);
}

int b200q_moe_mx4_linear(const void* W, const void* X, int x_dtype, int x_per_pair, const void* plan, const void* bias, void* Y, int y_dtype, int64_t tokens, int k,
                         int E, int N, int K, void* ws, size_t ws_bytes, void* stream) {
    return experts_common("moe_mx4_linear", W, nullptr, X, x_dtype, x_per_pair, plan, bias, Y, y_dtype, tokens, k, E, N, K, ws, ws_bytes, stream);
}

int b200q_moe_mx4_swiglu(const void* W_gate, const void* W_up, const void* X, int x_dtype, int x_per_pair, const void* plan, void* Y, int y_dtype, int64_t tokens, int k,
                         int E, int N, int K, void* ws, size_t ws_bytes, void* stream) {
    if (!W_up && tokens > 0 && N > 0) return fail(B200Q_ERR_BAD_ARG, "moe_mx4_swiglu: null pointer");
    return experts_common("moe_mx4_swiglu", W_gate, W_up, X, x_dtype, x_per_pair, plan, nullptr, Y, y_dtype, tokens, k, E, N, K, ws, ws_bytes, stream);
}

int b200q_moe_combine(const void* y, int dtype, const int32_t* ids, const float* weights, int64_t tokens, int k, int E, int N, void* out, void* stream) {
    if (!dtype_ok(dtype)) return fail(B200Q_ERR_BAD_ARG, "moe_combine: unknown dtype %d", dtype);
    if (tokens < 0 || N < 0 || k < 1 || E < 1) return fail(B200Q_ERR_BAD_ARG, "moe_combine: bad shape (tokens %lld, k %d, E %d, N %d)", (long long)tokens, k, E, N);
    if (tokens == 0 || N == 0) return B200Q_OK;
    if (!y || !ids || !weights || !out) return fail(B200Q_ERR_BAD_ARG, "moe_combine: null pointer");
    if (!on(y, dtype_size(dtype)) || !on(out, dtype_size(dtype)) || !on(ids, 4) || !on(weights, 4))
        return fail(B200Q_ERR_BAD_ARG, "moe_combine: pointers must be aligned to their elements");
    int sms, *status;
    if (int rc = device_facts(&sms, &status)) return rc;
    return launch_moe_combine(y, dtype, ids, weights, tokens, k, N, E, out, sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
