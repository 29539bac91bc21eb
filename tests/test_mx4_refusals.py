"""What the MXFP4 and expert entry points refuse, and what their sizes say, without a device: arguments are checked before it is touched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
import mx4_reference as ref

from brotensor_b200 import _capi as capi
from brotensor_b200 import ops


@pytest.fixture(scope="module")
def L():
    return capi.lib()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 8192)()
    yield (ctypes.addressof(buf) + 255) & ~255


BAD, UNSUP, WS, OK = capi.ERR_BAD_ARG, capi.ERR_UNSUPPORTED, capi.ERR_WORKSPACE, capi.OK


def test_sizes(L):
    assert L.b200q_mx4_image_bytes(1, 32) == L.b200q_mx4_image_bytes(128, 256) == 17408
    assert L.b200q_mx4_image_bytes(129, 256) == L.b200q_mx4_image_bytes(128, 288) == 2 * 17408
    assert L.b200q_mx4_image_bytes(0, 64) == 0 and L.b200q_mx4_image_bytes(4, 48) == 0 and L.b200q_mx4_image_bytes(-1, 32) == 0
    assert L.b200q_mx4_image_bytes(2 ** 33, 4096) == 2 ** 33 // 128 * 16 * 17408
    assert L.b200q_mx4_linear_workspace_bytes(300, 1024) == L.b200q_mx4_image_bytes(300, 1024)
    # up to 16 rows are quantised inside the product's launch, unless they are very long
    assert L.b200q_mx4_linear_workspace_bytes(16, 65536) == 0 and L.b200q_mx4_linear_workspace_bytes(17, 256) == 17408
    assert L.b200q_mx4_linear_workspace_bytes(1, 1 << 20) == L.b200q_mx4_image_bytes(1, 1 << 20)
    assert L.b200q_moe_mx4_workspace_bytes(2, 8, 64, 4096) == 0
    # tiles of 128 pairs: seventeen pairs at most seventeen; never more than pairs / 128 and one for each expert
    assert L.b200q_moe_mx4_workspace_bytes(17, 1, 64, 256) == 17 * 17408
    assert L.b200q_moe_mx4_workspace_bytes(3, 8, 4, 256) == 4 * 17408
    assert L.b200q_moe_mx4_workspace_bytes(512, 8, 64, 256) == (32 + 64) * 17408
    for t, k, e in ((-1, 1, 1), (1, 0, 4), (1, 33, 64), (1, 1, 0), (1, 1, 1025)):
        assert L.b200q_moe_plan_bytes(t, k, e) == 0 and L.b200q_moe_mx4_workspace_bytes(t, k, e, 256) == 0
    assert L.b200q_moe_plan_bytes(0, 2, 8) > 0


@pytest.mark.parametrize("pairs,E", [(1, 1), (5, 3), (128, 1), (129, 1), (130, 2), (1000, 7), (256, 300)])
def test_the_tiles_of_any_grouping_fit(L, pairs, E):
    """Every way to cut the groups that can need many tiles: one large group and single pairs, or groups of 128 i + 1."""
    L.b200q_set_option(b"mx4_few", 0)
    most = L.b200q_moe_mx4_workspace_bytes(pairs, 1, E, 256) // 17408
    L.b200q_set_option(b"mx4_few", 16)
    for met in range(1, min(E, pairs) + 1):
        sizes = [1] * (met - 1)
        left = pairs - (met - 1)
        for i in range(met - 1):
            if left - 128 >= 1:
                sizes[i] += 128
                left -= 128
        assert sum(-(-c // 128) for c in sizes + [left]) <= most


def test_mx4_arguments(L, p):
    f32 = capi.F32
    assert L.b200q_mx4_pack(p, 1, 4, 40, p, None) == BAD and b"multiple of 32" in L.b200q_last_error()
    assert L.b200q_mx4_pack(p, -1, 4, 32, p, None) == BAD and L.b200q_mx4_pack(None, 1, 4, 32, p, None) == BAD
    assert L.b200q_mx4_pack(p, 1, 4, 32, p + 8, None) == BAD and b"aligned" in L.b200q_last_error()
    assert L.b200q_mx4_pack(None, 0, 4, 32, None, None) == OK
    assert L.b200q_mx4_quantize(p, 9, 4, 32, p, None) == BAD and L.b200q_mx4_quantize(p, f32, 4, 0, p, None) == BAD
    assert L.b200q_mx4_quantize(p + 4, f32, 4, 32, p, None) == BAD and L.b200q_mx4_quantize(p, f32, -4, 32, p, None) == BAD
    assert L.b200q_mx4_quantize(None, f32, 0, 32, None, None) == OK
    assert L.b200q_mx4_dequantize(p, 4, 33, p, f32, None) == BAD and L.b200q_mx4_dequantize(p, 4, 32, p + 2, f32, None) == BAD
    assert L.b200q_mx4_dequantize(p, 4, 32, p, 2, None) == BAD and L.b200q_mx4_dequantize(None, 0, 32, None, f32, None) == OK
    g = lambda W=p, X=p, b=None, bt=f32, Y=p, yt=f32, M=1, N=4, K=32: L.b200q_mx4_gemm(W, X, b, bt, Y, yt, M, N, K, None)
    assert g(W=None) == BAD and g(X=p + 8) == BAD and g(Y=p + 2) == BAD and g(yt=3) == BAD and g(bt=7) == BAD
    assert g(b=p + 1, bt=capi.F16) == BAD and g(M=-1) == BAD and g(N=-1) == BAD and g(K=16) == BAD
    assert g(M=0) == OK and g(N=0) == OK and g(M=2 ** 30 + 1) == UNSUP
    lin = lambda X=p, ws=p, n=1 << 20, M=20, K=32, xt=f32: L.b200q_mx4_linear(p, X, xt, None, p, f32, M, 4, K, ws, n, None)
    assert lin(ws=None) == WS and lin(n=17407) == WS and lin(ws=p + 16) == WS and b"17408 bytes" in L.b200q_last_error()
    assert lin(X=p + 4) == BAD and lin(X=None) == BAD and lin(xt=5) == BAD and lin(K=8) == BAD and lin(M=-3) == BAD and lin(M=0, ws=None) == OK


def test_moe_arguments(L, p):
    f32 = capi.F32
    assert L.b200q_moe_plan(p, 4, 0, 8, p, None) == UNSUP and L.b200q_moe_plan(p, 4, 33, 64, p, None) == UNSUP
    assert L.b200q_moe_plan(p, 4, 2, 0, p, None) == UNSUP and L.b200q_moe_plan(p, 4, 2, 1025, p, None) == UNSUP
    assert L.b200q_moe_plan(p, -1, 2, 8, p, None) == BAD and L.b200q_moe_plan(None, 4, 2, 8, p, None) == BAD
    assert L.b200q_moe_plan(p, 4, 2, 8, p + 4, None) == BAD and L.b200q_moe_plan(p, 2 ** 30, 2, 8, p, None) == UNSUP
    r = lambda lg=p, dt=f32, T=4, E=8, k=2, ids=p, w=p, plan=p: L.b200q_moe_route(lg, dt, T, E, k, 1, 1.0, ids, w, plan, None)
    assert r(k=9) == BAD and b"more than E" in L.b200q_last_error()
    assert r(dt=3) == BAD and r(lg=None) == BAD and r(ids=None) == BAD and r(w=None) == BAD and r(lg=p + 2) == BAD and r(plan=p + 8) == BAD
    assert r(T=0, plan=None, lg=None) == OK
    m = lambda W=p, X=p, xt=f32, plan=p, b=None, Y=p, yt=f32, T=20, k=2, E=4, N=8, K=32, ws=p, n=1 << 30: L.b200q_moe_mx4_linear(
        W, X, xt, 0, plan, b, Y, yt, T, k, E, N, K, ws, n, None)
    assert m(W=None) == BAD and m(X=None) == BAD and m(plan=None) == BAD and m(Y=None) == BAD and m(xt=3) == BAD and m(yt=3) == BAD
    assert m(W=p + 8) == BAD and m(X=p + 8) == BAD and m(plan=p + 4) == BAD and m(Y=p + 1) == BAD and m(b=p + 2) == BAD
    assert m(K=40) == BAD and m(N=-1) == BAD and m(E=2000) == UNSUP and m(k=40) == UNSUP
    assert m(ws=None) == WS and m(n=4 * 17408 - 1) == WS and m(T=0, W=None, ws=None) == OK and m(N=0, ws=None) == OK
    assert L.b200q_moe_mx4_swiglu(p, None, p, f32, 0, p, p, f32, 2, 2, 4, 8, 32, p, 1 << 30, None) == BAD
    c = lambda y=p, dt=f32, ids=p, w=p, T=2, k=2, E=4, N=8, out=p: L.b200q_moe_combine(y, dt, ids, w, T, k, E, N, out, None)
    assert c(y=None) == BAD and c(out=None) == BAD and c(dt=3) == BAD and c(k=0) == BAD and c(E=0) == BAD and c(T=-1) == BAD
    assert c(y=p + 2) == BAD and c(ids=p + 2) == BAD and c(T=0, y=None) == OK and c(N=0) == OK


def test_python_front_end_refuses():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        ops.mx4_image_bytes(4, 40)
    with pytest.raises(ValueError):  # an image on the host
        ops.mx4_linear(torch.zeros(17408, dtype=torch.uint8), x, 4)
    with pytest.raises(ValueError):
        ops.mx4_pack(torch.zeros(17, dtype=torch.uint8), 1, 32)
    with pytest.raises(ValueError):
        ops.mx4_quantize(x.t())
    with pytest.raises(ValueError):
        ops.moe_route(x, 2)
    with pytest.raises(ValueError):
        ops.moe_plan(torch.zeros(4, 2, dtype=torch.int32), 8)
    with pytest.raises(ValueError):
        ops.moe_combine(torch.zeros(4, 2, 8), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))
    with pytest.raises(ValueError):
        ops.MoePlan(4, 2, 2000, "cpu")


def test_the_reference_quantises_as_the_format_says():
    """The test's own rule against values worked out by hand (amax 6.5 -> scale 1; midpoints to the even code)."""
    v = torch.zeros(1, 32)
    v[0, :14] = torch.tensor([6.5, 0.25, 0.26, 0.75, 1.25, 1.26, 1.75, 2.5, 2.6, 3.5, 5.0, 5.1, -5.0, -0.74])
    want = torch.zeros(1, 32, dtype=torch.float64)
    want[0, :14] = torch.tensor([6.0, 0.0, 0.5, 1.0, 1.0, 1.5, 2.0, 2.0, 3.0, 4.0, 4.0, 6.0, -4.0, -0.5])
    assert torch.equal(ref.quantise(v), want)
    assert torch.equal(ref.quantise(v * 2 ** -100), want * 2 ** -100)


def test_sizes_at_the_end_of_an_int(L):
    assert L.b200q_mx4_image_bytes(1, 2 ** 31 - 32) == 2 ** 23 * 17408 == ops.mx4_image_bytes(1, 2 ** 31 - 32)


def test_python_front_end_refuses_what_a_c_int_does_not_hold():
    """ctypes would pass the low 32 bits on, and a call with other sizes would be made."""
    with pytest.raises(ValueError, match="2\\^31"):
        ops.mx4_image_bytes(1, 2 ** 32 + 32)
    for k, experts in ((2, 2 ** 32 + 8), (2 ** 32 + 2, 8)):
        with pytest.raises(ValueError, match="supported sizes"):
            ops.MoePlan(1, k, experts, "cpu")
    for k, n, experts in ((1, 2 ** 32 + 8, 4), (2 ** 32 + 1, 8, 4), (1, 8, 2 ** 32 + 4)):
        with pytest.raises(ValueError, match="below 2"):
            ops.moe_combine(torch.empty(1, k, n, device="meta"), torch.empty(1, k, dtype=torch.int32, device="meta"), torch.empty(1, k, device="meta"), experts)
