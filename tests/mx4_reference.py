"""MXFP4 and sparse expert layers from their definitions, in 64 bits (torch, any device)."""
import torch

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def blocks_to_f64(blocks):
    """(..., 17) uint8 blocks (ggml block_mxfp4) -> (..., 32)."""
    b = blocks.long()
    q = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    lut = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device=blocks.device)
    scale = torch.exp2((b[..., :1] - 127).double())
    scale = torch.where(b[..., :1] == 255, torch.full_like(scale, float("nan")), scale)
    return lut[q] * scale


def matrix(blocks, rows, K):
    return blocks_to_f64(blocks.reshape(rows, K // 32, 17)).reshape(rows, K)


def quantise(x):
    """The values MXFP4 keeps of the rows of x: each element goes to the nearest value, the even code of two that are as near."""
    v = x.double().unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(v).all(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(torch.where(finite, top, torch.ones_like(top)))[1] - 3, -127).clamp(min=-127)
    scale = torch.exp2(e.double())
    a = (v / scale).abs().nan_to_num(0.0, 0.0, 0.0)
    lut = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    d = (a.unsqueeze(-1) - lut).abs()
    d[..., 1::2] += 1e-9  # (values and ties are multiples of 2^-26 of a scaled FP32: far coarser than this)
    q = lut[d.argmin(-1)]
    out = torch.copysign(q, v) * scale
    return torch.where(finite, out, torch.full_like(out, float("nan"))).flatten(-2)


def random_blocks(n, seed, lo=117, hi=121):
    g = torch.Generator().manual_seed(seed)
    b = torch.randint(0, 256, (n, 17), generator=g, dtype=torch.uint8)
    b[:, 0] = torch.randint(lo, hi, (n,), generator=g, dtype=torch.uint8)
    return b


def route(logits, k, normalize, scale):
    """ids, weights of each token; -inf and NaN are never chosen, ties go to the lower expert."""
    rows_i, rows_w = [], []
    for row in logits.double().cpu().tolist():
        cand = [(v, e) for e, v in enumerate(row) if v == v and v != float("-inf")]
        top = max((v for v, _ in cand), default=0.0)
        ex = {e: (1.0 if v == top else 0.0) if top == float("inf") else torch.exp(torch.tensor(v - top, dtype=torch.float64)).item() for v, e in cand}
        best = [e for _, e in sorted(cand, key=lambda c: (-c[0], c[1]))[:k]]
        total = sum(ex[e] for e in (best if normalize else ex))
        rows_i.append(best + [-1] * (k - len(best)))
        rows_w.append([scale * ex[e] / total for e in best] + [0.0] * (k - len(best)))
    return torch.tensor(rows_i, dtype=torch.int32).reshape(-1, k), torch.tensor(rows_w, dtype=torch.float64).reshape(-1, k)


def group(ids, E):
    """offsets (E + 1) and order (pairs, -1 behind the last) of a stable grouping."""
    groups = [[] for _ in range(E)]
    flat = ids.flatten().tolist()
    for s, e in enumerate(flat):
        if 0 <= e < E:
            groups[e].append(s)
    offsets, order = [0], []
    for g in groups:
        order += g
        offsets.append(len(order))
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(order + [-1] * (len(flat) - len(order)), dtype=torch.int32)
