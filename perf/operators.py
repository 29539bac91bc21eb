"""What the operators of sparse expert layers on 4-bit microscaled weights are measured on.

A block of a matrix in MXFP4 is 32 neighbouring elements of a row that share the scale 2^(e - 127); an element is one
of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (E2M1). Weights come from a file in blocks of 17 bytes - e, then 16 bytes whose
low nibbles are elements 0..15 and whose high nibbles are elements 16..31 - and are laid out once for the kernels.
Activations are quantised on the way: e - 127 = floor(log2(largest magnitude of the block)) - 2, elements rounded to
nearest, ties to even, magnitudes beyond 6 to 6.

A case is one of five kinds of pass:

  quantise  rows of a dense type to MXFP4 and back: the values the 4 bits stand for, in the type they came in.
  linear    y = quantise(x) W^T (+ bias), W in MXFP4: a projection.
  route     router logits -> the k best experts of each token (ties to the lower expert), their softmax weights, and the
            grouping of the token-expert pairs by expert: the first place of each expert and the pairs in that order.
  experts   each token's rows through the matrices of its k experts, ragged groups; `gated`: silu(gate) * up in one call.
  combine   the weighted sum of the k results of each token.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The activations of one decode step of six sequences.
        dict(name="quantise_step", kind="quantise", rows=6, k=4096, dtype="f16"),
        # A projection's weights converted at load or export.
        dict(name="quantise_weight", kind="quantise", rows=14336, k=4096, dtype="bf16"),
        # One user's chat: an up projection of one token.
        dict(name="linear_1", kind="linear", m=1, n=14336, k=4096, dtype="bf16", out="bf16", bias=False),
        # A chat turn of a few dozen tokens through a down projection, on a model whose widths are not powers of two.
        dict(name="linear_45", kind="linear", m=45, n=2560, k=6912, dtype="f32", out="f32", bias=True),
        # A long document's chunk.
        dict(name="linear_2000", kind="linear", m=2000, n=14336, k=4096, dtype="bf16", out="bf16", bias=False),
        # The router of one token.
        dict(name="route_1", kind="route", t=1, e=128, k=8, dtype="f32", normalize=True),
        # The router of a prefill chunk.
        dict(name="route_4096", kind="route", t=4096, e=64, k=6, dtype="bf16", normalize=False),
        # One token through the gated half of an expert layer.
        dict(name="experts_1", kind="experts", t=1, e=128, k=8, n=768, d=2048, dtype="bf16", out="bf16", gated=True, bias=False, per_slot=False),
        # A batch of decoding sequences through the second half: one row per token-expert pair, few rows per expert.
        dict(name="experts_96", kind="experts", t=96, e=64, k=6, n=2048, d=1408, dtype="f16", out="f16", gated=False, bias=True, per_slot=True),
        # A prefill chunk through the gated half.
        dict(name="experts_2000", kind="experts", t=2000, e=32, k=4, n=2048, d=4096, dtype="bf16", out="bf16", gated=True, bias=False, per_slot=False),
        # The results of one token put together: the smallest call.
        dict(name="combine_1", kind="combine", t=1, k=8, n=2048, dtype="f32"),
        # Those of a prefill chunk.
        dict(name="combine_2000", kind="combine", t=2000, k=8, n=2048, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(("quantise", "linear", "linear", "linear", "route", "experts", "experts", "experts", "combine"))
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    if kind == "quantise":
        k = 32 * max(1, round(_log(rng, 32, 14336) / 32))
        return dict(kind=kind, rows=max(1, int(_log(rng, 1, min(14336, 5.0e7 / k)))), k=k, dtype=dtype)
    if kind == "linear":
        n, k = int(_log(rng, 64, 16384)), 32 * round(_log(rng, 256, 14336) / 32)
        return dict(kind=kind, m=max(1, int(_log(rng, 1, min(2000, 1.1e11 / (n * k))))), n=n, k=k, dtype=dtype, out=rng.choice((dtype, "f32")),
                    bias=rng.random() < 0.4)
    e = rng.choice((8, 16, 32, 60, 64, 128, 160, 256))
    top = rng.randint(1, 8)
    if kind == "route":
        return dict(kind=kind, t=int(_log(rng, 1, 4096)), e=e, k=top, dtype=dtype, normalize=rng.random() < 0.6)
    if kind == "combine":
        return dict(kind=kind, t=int(_log(rng, 1, 2000)), k=top, n=int(_log(rng, 512, 8192 / top ** 0.5)), dtype=dtype)
    n, d = 8 * round(_log(rng, 256, 2048) / 8), 32 * round(_log(rng, 256, 4096) / 32)
    gated = rng.random() < 0.5
    e = max(8, min(e, int((3e8 if gated else 5e8) / (n * d))))
    return dict(kind=kind, t=int(_log(rng, 1, 2000)), e=e, k=top, n=n, d=d, dtype=dtype, out=rng.choice((dtype, "f32")), gated=gated,
                bias=not gated and rng.random() < 0.4, per_slot=not gated and rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------------------

class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def blocks(self, rows, k, scale=0):
        """Weights as a file holds them: uniform nibbles, scales 2^-10 .. 2^-7 (values of the order of 0.01)."""
        n = rows * (k // 32)
        b = torch.randint(-2 ** 31, 2 ** 31, ((n * 17 + 3) // 4,), dtype=torch.int32, device="cuda", generator=self.g).view(torch.uint8)[:n * 17].view(n, 17)
        b[:, 0] = torch.randint(117 + scale, 121 + scale, (n,), dtype=torch.uint8, device="cuda", generator=self.g)
        return b.view(rows, k // 32, 17)

    def normal(self, shape, dtype):
        """Activations: N(0, 1) with a few channels an order of magnitude larger."""
        x = torch.randn(shape, device="cuda", generator=self.g)
        x[..., torch.randint(0, shape[-1], (max(1, shape[-1] // 512),), device="cuda", generator=self.g)] *= 8
        return x.to(dtype)

    def logits(self, t, e, dtype):
        """Router logits: some experts are liked better than others."""
        liked = 0.7 * torch.randn(1, e, device="cuda", generator=self.g)
        return (torch.randn(t, e, device="cuda", generator=self.g) + liked).to(dtype)


def _inputs(case, seed):
    """What both forms start from: tensors by name."""
    d, kind = _Draw(seed), case["kind"]
    dt = _DT[case["dtype"]]
    if kind == "quantise":
        return dict(x=d.normal((case["rows"], case["k"]), dt))
    if kind == "linear":
        return dict(w=[d.blocks(case["n"], case["k"])], x=d.normal((case["m"], case["k"]), dt), b=d.normal((case["n"],), dt) if case["bias"] else None)
    if kind == "route":
        return dict(logits=d.logits(case["t"], case["e"], dt))
    t, k, n = case["t"], case["k"], case["n"]
    if kind == "combine":
        e = 4 * k
        ids = torch.rand(t, e, device="cuda", generator=d.g).argsort(1)[:, :k].int()
        return dict(y=d.normal((t, k, n), dt), ids=ids, weights=torch.rand(t, k, device="cuda", generator=d.g) / k)
    e, dim = case["e"], case["d"]
    return dict(w=[d.blocks(e * n, dim) for _ in range(2 if case["gated"] else 1)], x=d.normal((t, k, dim) if case["per_slot"] else (t, dim), dt),
                b=d.normal((e, n), dt) if case["bias"] else None,
                ids=d.logits(t, e, torch.float32).sort(dim=1, descending=True, stable=True)[1][:, :k].int())


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        from brotensor_b200 import ops
        s["ops"] = ops
        if case["kind"] == "linear":
            s["w"] = [ops.mx4_pack(w, case["n"], case["k"]) for w in s["w"]]
        elif case["kind"] == "experts":
            s["w"] = [ops.mx4_pack(w, case["n"], case["d"], count=case["e"]) for w in s["w"]]
            s["plan"] = ops.moe_plan(s["ids"], case["e"])
    elif case["kind"] in ("linear", "experts"):
        s["w"] = [_dense(w) for w in s["w"]]
        if case["kind"] == "experts":
            _groups(s, case)
    return s


def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s, s["case"])


# ---- the framework's operators ------------------------------------------------------------------------------

def _own_quantise(s, c):
    return s["ops"].mx4_dequantize(s["ops"].mx4_quantize(s["x"]), c["rows"], c["k"], out_dtype=s["x"].dtype)


def _own_linear(s, c):
    return s["ops"].mx4_linear(s["w"][0], s["x"], c["n"], bias=s["b"], out_dtype=_DT[c["out"]])


def _own_route(s, c):
    ids, weights, plan = s["ops"].moe_route(s["logits"], c["k"], normalize=c["normalize"])
    return ids, weights, plan.offsets, plan.order


def _own_experts(s, c):
    if c["gated"]:
        return s["ops"].moe_mx4_swiglu(s["w"][0], s["w"][1], s["x"], s["plan"], c["n"], out_dtype=_DT[c["out"]])
    return s["ops"].moe_mx4_linear(s["w"][0], s["x"], s["plan"], c["n"], bias=s["b"], out_dtype=_DT[c["out"]])


def _own_combine(s, c):
    return s["ops"].moe_combine(s["y"], s["ids"], s["weights"])


_own = dict(quantise=_own_quantise, linear=_own_linear, route=_own_route, experts=_own_experts, combine=_own_combine)


# ---- their plain form ---------------------------------------------------------------------------------------

def _dense(blocks):
    """Blocks of a file -> FP32."""
    rows, nb = blocks.shape[0], blocks.shape[1]
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    out = torch.empty(rows, nb * 32, device="cuda")
    step = max(1, (1 << 24) // (nb * 32))
    for r in range(0, rows, step):
        b = blocks[r:r + step].int()
        q = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
        out[r:r + step] = torch.ldexp(lut[q], b[..., :1] - 127).flatten(1)
    return out


def _quantise(x):
    """Rows -> the values that MXFP4 keeps of them, in FP32."""
    v = x.float().view(*x.shape[:-1], -1, 32)
    e = torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 3
    e = e.clamp(min=-127)
    a = torch.ldexp(v.abs(), -e)
    q = 0.5 * (a > 0.25) + 0.5 * (a >= 0.75) + 0.5 * (a > 1.25) + 0.5 * (a >= 1.75) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5)
    return torch.ldexp(torch.copysign(q, v), e).view(x.shape)


def _plain_quantise(s, c):
    return _quantise(s["x"]).to(s["x"].dtype)


def _plain_linear(s, c):
    y = _quantise(s["x"]) @ s["w"][0].T
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(_DT[c["out"]])


def _plain_route(s, c):
    logits = s["logits"].float()
    best, ids = logits.sort(dim=1, descending=True, stable=True)
    ids = ids[:, :c["k"]]
    e = torch.exp(best - best[:, :1])
    weights = e[:, :c["k"]] / (e[:, :c["k"]] if c["normalize"] else e).sum(1, keepdim=True)
    flat = ids.flatten()
    counts = (flat[None] == torch.arange(c["e"], device="cuda")[:, None]).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return ids.int(), weights, offsets.int(), flat.sort(stable=True)[1].int()


def _groups(s, c):
    """The pairs of each expert that has some. Few pairs each: a table of them, filled up to the longest group's length, for
    one batched product; many: an index per expert, for a product each."""
    flat = s["ids"].flatten().long()
    met, counts = flat.unique(return_counts=True)
    pairs = flat.sort(stable=True)[1]
    starts = counts.cumsum(0) - counts
    longest = int(counts.max())
    if longest > 128:
        s["groups"] = list(zip(met.tolist(), pairs.split(counts.tolist())))
        return
    s["met"] = met
    i = torch.arange(longest, device="cuda")
    s["table"] = pairs[starts[:, None] + torch.minimum(i[None], counts[:, None] - 1)]
    at = torch.empty_like(pairs)
    group = torch.repeat_interleave(torch.arange(len(met), device="cuda"), counts)
    at[pairs] = group * longest + torch.arange(len(pairs), device="cuda") - starts[group]
    s["at"] = at


def _plain_experts(s, c):
    n, d, k = c["n"], c["d"], c["k"]
    x = _quantise(s["x"]).reshape(-1, d)
    if "met" in s:
        xe = x[s["table"] if c["per_slot"] else s["table"] // k]
        r = [xe @ w.view(-1, n, d)[s["met"]].transpose(1, 2) for w in s["w"]]
        bias = None if s["b"] is None else s["b"][s["met"]][:, None]
        return _finished(r, bias, c).view(-1, n)[s["at"]].view(c["t"], k, n)
    y = torch.empty(c["t"] * k, n, dtype=_DT[c["out"]], device="cuda")
    for e, pairs in s["groups"]:
        xe = x[pairs if c["per_slot"] else pairs // k]
        r = [xe @ w[e * n:(e + 1) * n].T for w in s["w"]]
        y[pairs] = _finished(r, None if s["b"] is None else s["b"][e], c)
    return y.view(c["t"], k, n)


def _finished(r, bias, c):
    v = r[0] / (1 + torch.exp(-r[0])) * r[1] if c["gated"] else r[0] if bias is None else r[0] + bias.float()
    return v.to(_DT[c["out"]])


def _plain_combine(s, c):
    return (s["y"].float() * s["weights"][:, :, None]).sum(1).to(s["y"].dtype)


_plain = dict(quantise=_plain_quantise, linear=_plain_linear, route=_plain_route, experts=_plain_experts, combine=_plain_combine)


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------

def _dense64(blocks):
    b = blocks.long()
    q = torch.cat([b[..., 1:] % 16, b[..., 1:] // 16], -1)
    expo, man = (q % 8) // 2, (q % 2).double()
    mag = torch.where(expo == 0, man / 2, torch.exp2((expo - 1).double()) * (1 + man / 2))
    sign = 1.0 - 2.0 * (q // 8).double()
    return (sign * mag * torch.exp2((b[..., :1] - 127).double())).flatten(-2)


def _quantise64(x):
    v = x.double().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.where(top == 0, 2.0 ** -127, torch.exp2(torch.frexp(top)[1].double() - 3).clamp(min=2.0 ** -127))
    a = v / scale
    step = torch.exp2((torch.frexp(a)[1] - 1).clamp(min=0, max=2).double() - 1)  # half the power of two below the magnitude
    return ((a / step).round() * step).clamp(-6, 6).mul(scale).flatten(-2)


def _product64(x, blocks):
    rows = max(1, (1 << 25) // x.shape[1])
    return torch.cat([x @ _dense64(blocks[r:r + rows]).T for r in range(0, blocks.shape[0], rows)], 1)


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "quantise":
        return _quantise64(s["x"])
    if kind == "linear":
        y = _product64(_quantise64(s["x"]), s["w"][0])
        return y if s["b"] is None else y + s["b"].double()
    if kind == "combine":
        return torch.einsum("tkn,tk->tn", s["y"].double(), s["weights"].double())
    if kind == "route":
        logits = s["logits"].double().cpu()
        p = logits.softmax(1)
        ids = torch.tensor([sorted(range(case["e"]), key=lambda e: (-row[e], e))[:case["k"]] for row in logits.tolist()])
        weights = p.gather(1, ids)
        if case["normalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        groups = [[] for _ in range(case["e"])]
        for pair, e in enumerate(ids.flatten().tolist()):
            groups[e].append(pair)
        offsets = [0]
        for g in groups:
            offsets.append(offsets[-1] + len(g))
        return ids.int(), weights, torch.tensor(offsets, dtype=torch.int32), torch.tensor([p for g in groups for p in g], dtype=torch.int32)
    t, k, n, d = case["t"], case["k"], case["n"], case["d"]
    x = _quantise64(s["x"]).view(t, -1, d).expand(t, k, d)
    y = torch.empty(t, k, n, dtype=torch.float64, device="cuda")
    for e in range(case["e"]):
        mine = s["ids"] == e
        if not mine.any():
            continue
        r = [_product64(x[mine], w[e * n:(e + 1) * n]) for w in s["w"]]
        y[mine] = torch.nn.functional.silu(r[0]) * r[1] if case["gated"] else r[0] if s["b"] is None else r[0] + s["b"][e].double()
    return y


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    kind, size = case["kind"], _size(case["dtype"])
    if kind == "quantise":
        return {"bytes": 2 * size * case["rows"] * case["k"], "flops": 0}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k * 17 // 32 + size * (m * k + (n if case["bias"] else 0)) + _size(case["out"]) * m * n, "flops": 2 * m * n * k}
    t, k = case["t"], case["k"]
    if kind == "route":
        return {"bytes": size * t * case["e"] + 4 * (3 * t * k + case["e"] + 1), "flops": 0}
    n = case["n"]
    if kind == "combine":
        return {"bytes": size * (t * k * n + t * n) + 8 * t * k, "flops": 2 * t * k * n}
    e, d, mats = case["e"], case["d"], 2 if case["gated"] else 1
    met = e * (1 - (1 - k / e) ** t)  # experts that some token meets, were all liked alike
    return {"bytes": int(mats * met * n * d * 17 // 32) + size * (t * (k if case["per_slot"] else 1) * d + (int(met) * n if case["bias"] else 0)) + _size(case["out"]) * t * k * n,
            "flops": 2 * mats * t * k * n * d}
