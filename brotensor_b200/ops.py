"""Thin torch-tensor front end of the C-ABI, used by the tests and the benchmark.

Argument meaning follows brotensor's ops (include/brotensor/ops/quant.h): W is a
(N, K) quantized weight given as its raw GGUF block bytes, X is (M, K), the
result is (M, N). torch only supplies device memory and the current stream.
"""
from __future__ import annotations

import torch

from . import _capi as capi
from .synth import BLOCK_BYTES, BLOCK_ELEMS

_DT = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


# The current device's index and a device's current stream as plain integers: torch's own short cuts where this torch has them (they are not
# part of its public interface), else the public calls.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(t: torch.Tensor, f, *args) -> int:
    """f(*args, stream) with t's device current; the device is switched only when it is another one (entering and leaving
    torch.cuda.device and wrapping the stream in an object were a third of a small call's time on the host)."""
    i = t.get_device()  # -1: not on a CUDA device
    if i >= 0 and i == _current_device():
        return f(*args, _raw_stream(i))
    with torch.cuda.device(t.device):  # refuses a tensor that is not on a CUDA device
        return f(*args, _raw_stream(i))


def _check_w(fmt: int, W: torch.Tensor, N: int, K: int) -> None:
    if W.dtype != torch.uint8 or not W.is_cuda or not W.is_contiguous():
        raise ValueError("W must be a contiguous CUDA uint8 tensor holding raw GGUF blocks")
    if K % BLOCK_ELEMS[fmt]:
        raise ValueError(f"K ({K}) must be a multiple of {BLOCK_ELEMS[fmt]}")
    need = N * (K // BLOCK_ELEMS[fmt]) * BLOCK_BYTES[fmt]
    if W.numel() != need:
        raise ValueError(f"W holds {W.numel()} bytes, ({N}, {K}) needs {need}")


def repacked_fmt(fmt: int, K: int) -> int:
    """Format code of the device-side repacked form of raw format `fmt` for rows of K elements (`fmt` itself: none)."""
    return capi.lib().b200q_repacked_fmt(fmt, K)


def repack(fmt: int, W: torch.Tensor, N: int, K: int, inplace: bool = False) -> torch.Tensor:
    """Raw GGUF rows -> the layout the kernels read fastest (same size, bit-identical content)."""
    _check_w(fmt, W, N, K)
    out = W if inplace else torch.empty_like(W)
    capi.check(_launch(W, capi.lib().b200q_repack, fmt, W.data_ptr(), out.data_ptr(), N, K))
    return out


def unpack(fmt: int, W: torch.Tensor, N: int, K: int, inplace: bool = False) -> torch.Tensor:
    """Inverse of repack; `fmt` is the raw format."""
    _check_w(fmt, W, N, K)
    out = W if inplace else torch.empty_like(W)
    capi.check(_launch(W, capi.lib().b200q_unpack, fmt, W.data_ptr(), out.data_ptr(), N, K))
    return out


def dequant(fmt: int, W: torch.Tensor, N: int, K: int, out_dtype=torch.float16) -> torch.Tensor:
    _check_w(fmt, W, N, K)
    out = torch.empty((N, K), dtype=out_dtype, device=W.device)
    capi.check(_launch(W, capi.lib().b200q_dequant, fmt, W.data_ptr(), out.data_ptr(), _DT[out_dtype], N, K))
    return out


def embedding_gather(fmt: int, table: torch.Tensor, idx: torch.Tensor, rows: int, K: int, out_dtype=torch.float16) -> torch.Tensor:
    """out[b] = decode(table row idx[b]); idx: int32 device tensor. Rows outside the table come back as zeros."""
    _check_w(fmt, table, rows, K)
    if idx.dtype != torch.int32 or not idx.is_cuda or not idx.is_contiguous():
        raise ValueError("idx must be a contiguous CUDA int32 tensor")
    B = idx.numel()
    out = torch.empty((B, K), dtype=out_dtype, device=table.device)
    capi.check(_launch(table, capi.lib().b200q_embedding_gather, fmt, table.data_ptr(), idx.data_ptr(), B, rows, K, out.data_ptr(), _DT[out_dtype]))
    return out


def _linear(entry: str, fmt, W, X, N, bias, out, out_dtype, ws):
    if X.dim() == 1:
        X = X.unsqueeze(0)
    M, K = X.shape
    _check_w(fmt, W, N, K)
    if not X.is_contiguous():
        raise ValueError("X must be contiguous")
    if bias is not None and (bias.dtype != X.dtype or bias.numel() != N):
        raise ValueError("bias must have N elements of X's dtype")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or (torch.float16 if X.dtype == torch.float16 else torch.float32),
                          device=X.device)
    L = capi.lib()
    xt = _DT[X.dtype]
    args = (fmt, W.data_ptr(), X.data_ptr(), xt, bias.data_ptr() if bias is not None else None, out.data_ptr(), _DT[out.dtype], M, N, K)
    if entry == "gemv":
        capi.check(_launch(W, L.b200q_gemv, *args))
    elif entry == "gemm_static":
        capi.check(_launch(W, L.b200q_gemm_static, *args))
    else:
        if ws is None and M > 8:  # decode sizes need no workspace
            need = L.b200q_gemm_workspace_bytes(fmt, xt, M, N, K)
            if need:
                ws = torch.empty(need, dtype=torch.uint8, device=X.device)
        capi.check(_launch(W, L.b200q_gemm if entry == "gemm" else L.b200q_linear, *args, ws.data_ptr() if ws is not None else None,
                           ws.numel() if ws is not None else 0))
    return out


def gemv(fmt, W, X, N, bias=None, out=None, out_dtype=None):
    """Y(M,N) = X(M,K) @ decode(W).T (+bias), 1 <= M <= 8."""
    return _linear("gemv", fmt, W, X, N, bias, out, out_dtype, None)


def gemv_swiglu(fmt, W_gate, W_up, x, N, out=None, out_dtype=None):
    """y(1, N) = silu(x @ decode(W_gate).T) * (x @ decode(W_up).T) in one launch."""
    x = x.reshape(1, -1)
    K = x.shape[1]
    _check_w(fmt, W_gate, N, K)
    _check_w(fmt, W_up, N, K)
    if out is None:
        out = torch.empty((1, N), dtype=out_dtype or (torch.float16 if x.dtype == torch.float16 else torch.float32), device=x.device)
    capi.check(_launch(x, capi.lib().b200q_gemv_swiglu, fmt, W_gate.data_ptr(), W_up.data_ptr(), x.data_ptr(), _DT[x.dtype],
                       out.data_ptr(), _DT[out.dtype], N, K))
    return out


def gemv_multi(fmt, Ws, x, Ns, outs=None, biases=None):
    """Several matrices against one activation vector in one launch; returns the list of (1, N_s) results."""
    import ctypes as C
    n = len(Ws)
    K = x.numel()
    for W, N in zip(Ws, Ns):
        _check_w(fmt, W, N, K)
    if outs is None:
        outs = [torch.empty((1, N), dtype=torch.float32, device=x.device) for N in Ns]
    Wp = (C.c_void_p * n)(*[W.data_ptr() for W in Ws])
    Yp = (C.c_void_p * n)(*[y.data_ptr() for y in outs])
    Np = (C.c_int * n)(*Ns)
    Bp = None if biases is None else (C.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in biases])
    capi.check(_launch(x, capi.lib().b200q_gemv_multi, fmt, n, Wp, Np, Yp, Bp, x.data_ptr(), _DT[x.dtype], _DT[outs[0].dtype], K))
    return outs


def gemv_multi_rmsnorm(fmt, Ws, x, gamma, eps, Ns, outs=None):
    """gemv_multi on rms_norm(x) * gamma, the normalisation folded into the kernel."""
    import ctypes as C
    n = len(Ws)
    K = x.numel()
    for W, N in zip(Ws, Ns):
        _check_w(fmt, W, N, K)
    if gamma.dtype != x.dtype or gamma.numel() != K:
        raise ValueError("gamma must have K elements of x's dtype")
    if outs is None:
        outs = [torch.empty((1, N), dtype=torch.float32, device=x.device) for N in Ns]
    Wp = (C.c_void_p * n)(*[W.data_ptr() for W in Ws])
    Yp = (C.c_void_p * n)(*[y.data_ptr() for y in outs])
    Np = (C.c_int * n)(*Ns)
    capi.check(_launch(x, capi.lib().b200q_gemv_multi_rmsnorm, fmt, n, Wp, Np, Yp, None, x.data_ptr(), _DT[x.dtype], gamma.data_ptr(), float(eps),
                       _DT[outs[0].dtype], K))
    return outs


def gemm(fmt, W, X, N, bias=None, out=None, out_dtype=None, ws=None):
    """Prefill GEMM on the tensor cores, any M."""
    return _linear("gemm", fmt, W, X, N, bias, out, out_dtype, ws)


def gemm_static(fmt, W, X, N, bias=None, out=None, out_dtype=None):
    """The GEMM with its scratch in the library's fixed device array: makes no allocation."""
    return _linear("gemm_static", fmt, W, X, N, bias, out, out_dtype, None)


def linear(fmt, W, X, N, bias=None, out=None, out_dtype=None, ws=None):
    """Routing of the batched ops: M <= 8 -> gemv, else gemm."""
    return _linear("linear", fmt, W, X, N, bias, out, out_dtype, ws)


# ---- MXFP4 matrices and sparse expert layers on them -------------------------------------------------------

# (The wrappers below are written for short calls: a decode step makes a dozen of them per layer, and at a few microseconds each every call on the
# way counts. They look at everything in one condition and go to the checks that say what is wrong only where it fails.)

def mx4_image_bytes(rows: int, K: int) -> int:
    """Bytes of the image of a rows x K matrix in MXFP4 (K a multiple of 32)."""
    if rows < 0 or K <= 0 or K % 32 or K >> 31:
        raise ValueError(f"K ({K}) must be a positive multiple of 32 below 2^31")
    return ((rows + 127) >> 7) * ((K + 255) >> 8) * 17408


def _check_image(W: torch.Tensor, rows: int, K: int, count: int = 1) -> int:
    """Returns the device index of an image that is one."""
    device = W.get_device()
    if device < 0 or W.dtype != torch.uint8 or not W.is_contiguous():
        raise ValueError("an image is a contiguous CUDA uint8 tensor (mx4_pack, mx4_quantize)")
    if W.numel() < count * mx4_image_bytes(rows, K):
        raise ValueError(f"the image holds {W.numel()} bytes, {count} x ({rows}, {K}) needs {count * mx4_image_bytes(rows, K)}")
    return device


def _is_image(W: torch.Tensor, rows: int, K: int, count: int, device: int) -> bool:
    return (W.dtype is torch.uint8 and W.get_device() == device >= 0 and 0 < K < 2 ** 31 and not K & 31 and rows >= 0 and W.is_contiguous()
            and W.numel() >= count * ((rows + 127) >> 7) * ((K + 255) >> 8) * 17408)


def _check_dense(t: torch.Tensor, what: str, device: int) -> int:
    """Returns the type code of a contiguous tensor of one of the dense types on device `device`."""
    code = _DT.get(t.dtype)
    if code is None or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32, float16 or bfloat16 tensor")
    if t.get_device() != device or device < 0:
        raise ValueError(f"{what} is on {t.device}, not on CUDA device {device}")
    return code


def _check_int32(t: torch.Tensor, what: str, shape, device: int) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)}")
    if t.get_device() != device or device < 0:
        raise ValueError(f"{what} is on {t.device}, not on CUDA device {device}")


def _check_out(out: torch.Tensor, shape, out_dtype, device: int) -> None:
    if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out must be of shape {tuple(shape)}" + (f" and {out_dtype}" if out_dtype is not None else ""))
    _check_dense(out, "out", device)


def _default_out(x: torch.Tensor) -> torch.dtype:
    return torch.float16 if x.dtype == torch.float16 else torch.float32


def _scratch(ws, need: int, x: torch.Tensor):
    """(pointer, bytes) of the workspace, made here where the caller gives none; and the tensor, to be kept until the call is made."""
    if ws is None:
        if not need:
            return None, 0, None
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    elif ws.dtype != torch.uint8 or not ws.is_contiguous() or ws.device != x.device:
        raise ValueError(f"ws must be a contiguous uint8 tensor on {x.device}")
    return ws.data_ptr(), ws.numel(), ws


def mx4_pack(blocks: torch.Tensor, rows: int, K: int, count: int = 1, out=None) -> torch.Tensor:
    """A file's MXFP4 blocks of `count` matrices of rows x K -> their images, one after the other."""
    if blocks.dtype != torch.uint8 or not blocks.is_cuda or not blocks.is_contiguous():
        raise ValueError("blocks must be a contiguous CUDA uint8 tensor")
    size = mx4_image_bytes(rows, K)
    if count < 0 or blocks.numel() != count * rows * (K // 32) * 17:
        raise ValueError(f"blocks hold {blocks.numel()} bytes, {count} x ({rows}, {K}) needs {count * rows * (K // 32) * 17}")
    if out is None:
        out = torch.empty(count * size, dtype=torch.uint8, device=blocks.device)
    elif _check_image(out, rows, K, count) != blocks.get_device():
        raise ValueError("out is on another device than the blocks")
    capi.check(_launch(blocks, capi.lib().b200q_mx4_pack, blocks.data_ptr(), count, rows, K, out.data_ptr()))
    return out


def mx4_quantize(x: torch.Tensor, out=None) -> torch.Tensor:
    """(rows, K) float32 / float16 / bfloat16 -> image."""
    if x.dim() != 2:
        raise ValueError("x must be (rows, K)")
    device, code = x.get_device(), _DT.get(x.dtype)
    if code is None or device < 0 or not x.is_contiguous():
        _check_dense(x, "x", device)
    rows, K = x.shape
    size = mx4_image_bytes(rows, K)
    if out is None:
        out = torch.empty(size, dtype=torch.uint8, device=x.device)
    elif _check_image(out, rows, K) != device:
        raise ValueError("out is on another device than x")
    capi.check(_launch(x, capi.lib().b200q_mx4_quantize, x.data_ptr(), code, rows, K, out.data_ptr()))
    return out


def mx4_dequantize(image: torch.Tensor, rows: int, K: int, out_dtype=torch.float32) -> torch.Tensor:
    """The values of an image, (rows, K)."""
    if not _is_image(image, rows, K, 1, image.get_device()):
        _check_image(image, rows, K)
    code = _DT.get(out_dtype)
    if code is None:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    out = torch.empty(rows, K, dtype=out_dtype, device=image.device)
    capi.check(_launch(image, capi.lib().b200q_mx4_dequantize, image.data_ptr(), rows, K, out.data_ptr(), code))
    return out


def mx4_gemm(W: torch.Tensor, X: torch.Tensor, M: int, N: int, K: int, bias=None, out=None, out_dtype=None) -> torch.Tensor:
    """Y(M,N) = X(M,K) @ W(N,K).T (+bias) of two images; float32 unless out_dtype says otherwise."""
    device = _check_image(W, N, K)
    if _check_image(X, M, K) != device:
        raise ValueError("W and X are on different devices")
    bias_code = capi.F32
    if bias is not None:
        bias_code = _check_dense(bias, "bias", device)
        if bias.numel() != N:
            raise ValueError("bias must have N elements")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or torch.float32, device=W.device)
    else:
        _check_out(out, (M, N), out_dtype, device)
    capi.check(_launch(W, capi.lib().b200q_mx4_gemm, W.data_ptr(), X.data_ptr(), bias.data_ptr() if bias is not None else None, bias_code,
                       out.data_ptr(), _DT[out.dtype], M, N, K))
    return out


def mx4_linear(W: torch.Tensor, X: torch.Tensor, N: int, bias=None, out=None, out_dtype=None, ws=None) -> torch.Tensor:
    """Y(M,N) = quantise(X(M,K)) @ W(N,K).T (+bias), W an image, X float32 / float16 / bfloat16."""
    if X.dim() == 1:
        X = X.unsqueeze(0)
    if X.dim() != 2:
        raise ValueError("X must be (M, K)")
    M, K = X.shape
    device, code = X.get_device(), _DT.get(X.dtype)
    if code is None or not X.is_contiguous() or not _is_image(W, N, K, 1, device):
        _check_dense(X, "X", _check_image(W, N, K))
        raise ValueError("W and X are on different devices")
    bias_ptr = None
    if bias is not None:
        if _check_dense(bias, "bias", device) != code or bias.numel() != N:
            raise ValueError("bias must have N elements of X's dtype")
        bias_ptr = bias.data_ptr()
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype or _default_out(X), device=X.device)
    else:
        _check_out(out, (M, N), out_dtype, device)
    L = capi.lib()
    need = L.b200q_mx4_linear_workspace_bytes(M, K)
    ws_ptr, ws_bytes, ws = _scratch(ws, need, X) if need or ws is not None else (None, 0, None)
    capi.check(_launch(X, L.b200q_mx4_linear, W.data_ptr(), X.data_ptr(), code, bias_ptr, out.data_ptr(), _DT[out.dtype], M, N, K, ws_ptr, ws_bytes))
    return out


class MoePlan:
    """The pairs of tokens and experts grouped by expert. offsets (E + 1) and order (tokens * k): expert e has the pairs
    order[offsets[e]:offsets[e + 1]], in their own order; pair s = t * k + j is token t's j-th choice. Device tensors, int32."""

    __slots__ = ("tokens", "k", "experts", "data")

    def __init__(self, tokens: int, k: int, experts: int, device):
        size = capi.lib().b200q_moe_plan_bytes(tokens, k, experts) if 0 < k <= 32 and 0 < experts <= 1024 else 0  # (a C int holds no more than 31 bits)
        if not size:
            raise ValueError(f"{tokens} tokens, {k} of {experts} experts each: outside the supported sizes (1..1024 experts, 1..32 each)")
        self.tokens, self.k, self.experts = tokens, k, experts
        self.data = torch.empty(size >> 2, dtype=torch.int32, device=device)

    @property
    def offsets(self) -> torch.Tensor:
        return self.data.as_strided((self.experts + 1,), (1,), 0)

    @property
    def order(self) -> torch.Tensor:
        return self.data.as_strided((self.tokens * self.k,), (1,), self.experts + 1)


def moe_plan(ids: torch.Tensor, experts: int) -> MoePlan:
    """Groups (tokens, k) int32 expert ids by expert. An id outside 0 .. experts - 1 is no expert."""
    if ids.dim() != 2:
        raise ValueError("ids must be a (tokens, k) CUDA tensor")
    _check_int32(ids, "ids", ids.shape, ids.get_device())
    plan = MoePlan(ids.shape[0], ids.shape[1], experts, ids.device)
    capi.check(_launch(ids, capi.lib().b200q_moe_plan, ids.data_ptr(), plan.tokens, plan.k, experts, plan.data.data_ptr()))
    return plan


def moe_route(logits: torch.Tensor, k: int, normalize: bool = True, scale: float = 1.0):
    """(tokens, E) logits -> (ids, weights, plan): the k best experts of each token, ties to the lower one; their softmax
    weights over the chosen (normalize) or over all experts, times scale; the grouping by expert."""
    if logits.dim() != 2:
        raise ValueError("logits must be a (tokens, E) CUDA tensor")
    code = _DT.get(logits.dtype)
    if code is None or logits.get_device() < 0 or not logits.is_contiguous():
        _check_dense(logits, "logits", logits.get_device())
    T, E = logits.shape
    device = logits.device
    plan = MoePlan(T, k, E, device)
    ids = torch.empty(T, k, dtype=torch.int32, device=device)
    weights = torch.empty(T, k, dtype=torch.float32, device=device)
    capi.check(_launch(logits, capi.lib().b200q_moe_route, logits.data_ptr(), code, T, E, k, 1 if normalize else 0, scale, ids.data_ptr(),
                       weights.data_ptr(), plan.data.data_ptr()))
    return ids, weights, plan


def _moe_common(Ws, X, plan, N, out, out_dtype, ws):
    """Checks; returns (type code of X, 1 if X has a row per pair, out, K, workspace)."""
    T, k, E = plan.tokens, plan.k, plan.experts
    shape = X.shape
    if (len(shape) != 2 and (len(shape) != 3 or shape[1] != k)) or shape[0] != T:
        raise ValueError(f"X must be ({T}, K) or ({T}, {k}, K), as the plan")
    device, K, code = plan.data.get_device(), shape[-1], _DT.get(X.dtype)
    if code is None or X.get_device() != device or not X.is_contiguous():
        _check_dense(X, "X", device)
    for W in Ws:
        if not _is_image(W, N, K, E, device):
            _check_image(W, N, K, E)
            raise ValueError("the weights are on another device than X")
    if out is None:
        out = torch.empty(T, k, N, dtype=out_dtype or _default_out(X), device=X.device)
    else:
        _check_out(out, (T, k, N), out_dtype, device)
    need = capi.lib().b200q_moe_mx4_workspace_bytes(T, k, E, K)
    return code, len(shape) - 2, out, K, _scratch(ws, need, X) if need or ws is not None else (None, 0, None)


def moe_mx4_linear(W, X, plan: MoePlan, N: int, bias=None, out=None, out_dtype=None, ws=None) -> torch.Tensor:
    """out[t][j] = quantise(X[t] or X[t][j]) @ W[e].T (+ bias[e]), e the j-th expert of token t: (tokens, k, N). W: the
    experts' images, one after the other. Rows of pairs without an expert are left as they were: in an `out` made here they hold
    whatever the memory held (moe_combine and a further product do not read them; other operations would)."""
    code, per_pair, out, K, (ws_ptr, ws_bytes, ws) = _moe_common((W,), X, plan, N, out, out_dtype, ws)
    bias_ptr = None
    if bias is not None:
        if _check_dense(bias, "bias", X.get_device()) != code or bias.shape != (plan.experts, N):
            raise ValueError("bias must be (experts, N) of X's dtype")
        bias_ptr = bias.data_ptr()
    capi.check(_launch(X, capi.lib().b200q_moe_mx4_linear, W.data_ptr(), X.data_ptr(), code, per_pair, plan.data.data_ptr(), bias_ptr, out.data_ptr(),
                       _DT[out.dtype], plan.tokens, plan.k, plan.experts, N, K, ws_ptr, ws_bytes))
    return out


def moe_mx4_swiglu(W_gate, W_up, X, plan: MoePlan, N: int, out=None, out_dtype=None, ws=None) -> torch.Tensor:
    """silu(gate) * up of the two products, without writing them out. Rows of pairs without an expert: as moe_mx4_linear."""
    code, per_pair, out, K, (ws_ptr, ws_bytes, ws) = _moe_common((W_gate, W_up), X, plan, N, out, out_dtype, ws)
    capi.check(_launch(X, capi.lib().b200q_moe_mx4_swiglu, W_gate.data_ptr(), W_up.data_ptr(), X.data_ptr(), code, per_pair, plan.data.data_ptr(),
                       out.data_ptr(), _DT[out.dtype], plan.tokens, plan.k, plan.experts, N, K, ws_ptr, ws_bytes))
    return out


def moe_combine(y: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, experts: int = 2 ** 31 - 1, out=None) -> torch.Tensor:
    """out[t] = sum_j weights[t][j] * y[t][j]; pairs whose id is negative (or not below `experts`) are left out."""
    if y.dim() != 3:
        raise ValueError("y must be a (tokens, k, N) CUDA tensor")
    T, k, N = y.shape
    if k >> 31 or N >> 31 or experts >= 1 << 31:
        raise ValueError(f"k ({k}), N ({N}) and experts ({experts}) must be below 2^31")
    if experts < 1:
        raise ValueError(f"experts ({experts}) must be positive")
    device, code, pairs = y.get_device(), _DT.get(y.dtype), (T, k)
    if (code is None or device < 0 or ids.dtype is not torch.int32 or weights.dtype is not torch.float32 or ids.shape != pairs or weights.shape != pairs
            or ids.get_device() != device or weights.get_device() != device or not (y.is_contiguous() and ids.is_contiguous() and weights.is_contiguous())):
        _check_dense(y, "y", device)
        _check_int32(ids, "ids", pairs, device)
        raise ValueError(f"weights must be a contiguous float32 tensor of shape {pairs} on {y.device}")
    if out is None:
        out = torch.empty(T, N, dtype=y.dtype, device=y.device)
    else:
        _check_out(out, (T, N), y.dtype, device)
    capi.check(_launch(y, capi.lib().b200q_moe_combine, y.data_ptr(), code, ids.data_ptr(), weights.data_ptr(), T, k, experts, N, out.data_ptr()))
    return out


def set_option(key: str, value: int) -> None:
    capi.check(capi.lib().b200q_set_option(key.encode(), value))


def get_option(key: str) -> int:
    import ctypes
    v = ctypes.c_int(0)
    capi.check(capi.lib().b200q_get_option(key.encode(), ctypes.byref(v)))
    return v.value


def device_status() -> int:
    """Synchronises; returns 0 or raises if a kernel's bounded wait ran out."""
    import ctypes
    v = ctypes.c_int(0)
    capi.check(capi.lib().b200q_device_status(ctypes.byref(v)))
    return v.value


def tc_calls_consume(fmt: int) -> int:
    return int(capi.lib().b200q_tc_calls_consume(fmt))
