"""silu(gate) * up over the whole range of gates, far negative ones beside large ups among them."""
import pytest

torch = pytest.importorskip("torch")
import mx4_exact as exact
import mx4_reference as ref
from test_gpu_mx4 import F32, route  # noqa: F401

from brotensor_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("up_scale", [0, 100])
@pytest.mark.parametrize("T", [8, 200])
def test_silu_times_up(T, up_scale, route):
    """Both products are exact (mx4_exact.py; a power of two on the second). exp(-|g| / 2), taken twice, within 2^-22 each time, a reciprocal within 2^-23, a sum and five
    products: 4.5 units of 2^-22; the rounded argument of the exponential |g| 2^-24 more, of the exponential. Where silu(g) lies below 2^-126 its unit is 2^-149, and up
    multiplies that."""
    N, K = 2048, 64
    bg, bu = exact.weights(N, K, 1).cuda(), exact.weights(N, K, 2).cuda()
    bu[:, 0] += up_scale
    G, U = (ops.mx4_pack(b.reshape(-1), N, K) for b in (bg, bu))
    x = exact.activations((T, K), F32, 3, device="cuda")
    g, u = (x.double() @ ref.matrix(b, N, K).T for b in (bg, bu))
    assert int(((g < -87.5) & (g > -88.5) & (u != 0)).sum()) > 20 and g.max() > 100
    want = g / (1 + torch.exp(-g)) * u
    got = ops.moe_mx4_swiglu(G, U, x, ops.moe_plan(torch.zeros(T, 1, dtype=torch.int32, device="cuda"), 1), N, out_dtype=F32)[:, 0].double()
    bound = want.abs() * (4.5 * 2.0 ** -22 + (-g).clamp(min=0) * 2.0 ** -24 + 2.0 ** -24) + u.abs() * 2.0 ** -148 + 2.0 ** -149
    off = (got - want).abs()
    assert (off <= bound).all(), f"{int((off > bound).sum())} off, at gates {g[off > bound][:4].tolist()}: {got[off > bound][:4].tolist()} for {want[off > bound][:4].tolist()}"
