// MXFP4 weights and sparse expert layers on them (b200q.h: b200q_mx4_*, b200q_moe_*). Not in brotensor, whose loader does not
// know the format and whose op table has no expert layer; shapes and errors follow the conventions of ops/quant.h.
//
// A weight as a file holds it is a Tensor of Dtype::MXFP4 (gguf::File hands out such tensors); the ops take its image, made once by
// mxfp4_pack: a Tensor of Dtype::INT8 with one row per tile of 128 x 256 elements; of Dtype::INT32, with as many rows, from 2^31 bytes on, up to 2^31 words (8.6 GB). Activations are FP32, FP16 or BF16, quantised on the way. Results
// keep a pre-sized FP32 / FP16 / BF16 destination of the right shape, else they are FP16 for FP16 activations and FP32 for the others.
// Scratch comes from the stream-ordered pool, so that every op may be captured.
#pragma once

#include "../tensor.h"

namespace brotensor_b200 {

// W (experts * out, in) -> image of `experts` matrices of (out, in), one after the other.
void mxfp4_pack(const Tensor& W, int experts, Tensor& image);
// Y (B, out) = X (B, in) W^T (+ bias, `out` values of X's dtype)
void mxfp4_linear_forward(const Tensor& image, int out, const Tensor* bias, const Tensor& X_BD, Tensor& Y_BD);

// The k best experts of each token, largest logit first, ties to the lower one: ids (T, k) INT32, -1 where none is left, and FP32 softmax weights
// over the chosen (normalize) or over all experts, times scale; plan: INT32, the grouping of the T * k pairs by expert.
void moe_route_forward(const Tensor& logits_TE, int k, bool normalize, float scale, Tensor& ids, Tensor& weights, Tensor& plan);
// Y (T * k, out): row t * k + j is token t's row of X through its j-th expert. X: (T, in), or (T * k, in) with a row for each pair. Rows of pairs without
// an expert are left as they were (uninitialised where Y is made or resized here; moe_combine_forward and a further product do not read them). bias: (experts, out) of X's dtype or nullptr.
void moe_linear_forward(const Tensor& image, int experts, int out, const Tensor* bias, const Tensor& X, const Tensor& plan, int tokens, int k, Tensor& Y);
// silu(gate) * up of two such products
void moe_swiglu_forward(const Tensor& gate_image, const Tensor& up_image, int experts, int out, const Tensor& X, const Tensor& plan, int tokens, int k, Tensor& Y);
// out (T, N) = weighted sum over the k rows of each token; Y (T * k, N), out of Y's dtype
void moe_combine_forward(const Tensor& Y, const Tensor& ids, const Tensor& weights, int experts, Tensor& out);

}  // namespace brotensor_b200
