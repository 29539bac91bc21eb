"""Sparse expert layers on MXFP4 weights on the B200: routing, grouping, grouped products and their sum, against the definitions
in 64 bits. Tolerances of the products as in test_gpu_mx4.py; softmax weights are a quotient of FP32 sums of at most E terms whose exp is
within 2 units of the last place (2^-22) of an argument that one subtraction has rounded (|l - max| 2^-24 relative)."""
import pytest

torch = pytest.importorskip("torch")
import mx4_reference as ref
from test_gpu_mx4 import BF16, F16, F32, _check, _randn, _weights, route  # noqa: F401

from brotensor_b200 import ops

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _ids(T, k, E, seed, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    p = torch.randn(E, generator=g).exp()
    ids = torch.multinomial(p.expand(T, E), k, generator=g).int() if T else torch.zeros(0, k, dtype=torch.int32)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    return ids


def _check_plan(plan, ids, E):
    offsets, order = ref.group(ids, E)
    assert torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(plan.order.cpu(), order)


def _check_route(logits, k, normalize, scale=1.0):
    ids, weights, plan = ops.moe_route(logits, k, normalize=normalize, scale=scale)
    want_ids, want = ref.route(logits, k, normalize, scale)
    assert torch.equal(ids.cpu(), want_ids)
    E = logits.shape[1]
    spread = float((logits.double() - logits.double().nan_to_num(0, 0, 0).amax(1, keepdim=True)).abs().nan_to_num(0, 0, 0).max()) if logits.numel() else 0
    assert ((weights.cpu().double() - want).abs() <= want * ((E + 8) * 2.0 ** -24 + 2 * (2.0 ** -22 + spread * 2.0 ** -24)) + 1e-37).all()
    _check_plan(plan, want_ids, E)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 8), (5, 7, 7), (33, 60, 4), (300, 256, 8), (129, 1000, 32), (700, 64, 6), (2100, 16, 2)])
def test_route(T, E, k, normalize, dtype):
    _check_route(_randn((T, E), dtype, T + E), k, normalize, 2.5)


def test_route_ties_and_masks():
    x = torch.zeros(12, 40)
    x[1] = -0.0
    x[1, 3:9] = 0.0
    x[2, 5:] = -INF
    x[3] = -INF
    x[4] = NAN
    x[5, ::2] = NAN
    x[6, 11] = INF
    x[7, [4, 30]] = INF
    x[8] = torch.finfo(F32).min
    x[9, 1] = torch.finfo(F32).max
    x[10] = -1e30
    x[10, 39] = -INF
    x[11, 20:] = torch.finfo(F32).min
    for normalize in (True, False):
        _check_route(x.cuda(), 6, normalize)
        _check_route(x.cuda().to(BF16), 6, normalize)


@pytest.mark.parametrize("T,k,E,drop", [(1, 1, 1, 0), (1, 8, 128, 0), (100, 8, 16, 0.3), (1024, 1, 8, 0), (1025, 1, 3, 0), (513, 2, 1000, 0.1), (3000, 8, 60, 0.02), (40000, 4, 256, 0)])
def test_plan(T, k, E, drop):
    ids = _ids(T, k, max(E, k), T + E, drop)
    _check_plan(ops.moe_plan(ids.cuda(), E), ids, E)  # (ids from E on are no expert)


def test_plan_odd_ids():
    ids = torch.tensor([[3, 3, 3], [-1, 7, 2 ** 31 - 1], [-2 ** 31, 0, 8], [5, 5, 0]], dtype=torch.int32)
    _check_plan(ops.moe_plan(ids.cuda(), 8), ids, 8)
    none = torch.full((50, 2), -1, dtype=torch.int32)
    _check_plan(ops.moe_plan(none.cuda(), 4), none, 4)
    empty = torch.zeros(0, 3, dtype=torch.int32)
    _check_plan(ops.moe_plan(empty.cuda(), 4), empty, 4)


def _products(Ws, x, ids, N, bias=None):
    """want, sum |a b| of every pair (zeros where there is no expert)."""
    T, k = ids.shape
    q = ref.quantise(x)
    q = q if x.dim() == 3 else q[:, None].expand(T, k, -1)
    e = ids.long().cuda().clamp(0, Ws[0].shape[0] - 1)
    out = []
    for w in Ws:
        y, s = torch.zeros(T, k, N, dtype=torch.float64, device="cuda"), torch.zeros(T, k, N, dtype=torch.float64, device="cuda")
        for i in range(w.shape[0]):
            m = e == i
            y[m], s[m] = q[m] @ w[i].T, q[m].abs() @ w[i].abs().T
        out.append((y, s))
    return out, e


@pytest.mark.parametrize("per_pair", [False, True])
@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 32, 32), (1, 8, 128, 256, 512), (3, 2, 8, 77, 96), (50, 4, 16, 200, 544), (300, 2, 3, 130, 256), (96, 6, 64, 384, 1408), (700, 4, 5, 128, 320)])
def test_experts(T, k, E, N, K, per_pair, route):
    W, w = _weights(N, K, N + K, count=E)
    ids = _ids(T, k, E, T) if k <= E else torch.zeros(T, k, dtype=torch.int32)
    x = _randn((T, k, K) if per_pair else (T, K), BF16, 3)
    plan = ops.moe_plan(ids.cuda(), E)
    ((want, terms),), _ = _products([w], x, ids, N)
    got = ops.moe_mx4_linear(W, x, plan, N, out_dtype=F32)
    _check(got, want, terms, K)
    assert torch.equal(got, ops.moe_mx4_linear(W, x, plan, N, out_dtype=F32)), "the same call gives other bits"


@pytest.mark.parametrize("x_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("y_dtype", [F32, F16, BF16])
def test_experts_bias_types_and_pairs_without_an_expert(x_dtype, y_dtype, route):
    T, k, E, N, K = 40, 3, 6, 150, 288
    W, w = _weights(N, K, 5, count=E)
    ids = _ids(T, k, E, 6, drop=0.25)
    ids[4] = -1
    ids[5] = torch.tensor([2, 2, 9])
    x, b = _randn((T, K), x_dtype, 7), _randn((E, N), x_dtype, 8)
    out = torch.full((T, k, N), 77.0, dtype=y_dtype, device="cuda")
    got = ops.moe_mx4_linear(W, x, ops.moe_plan(ids.cuda(), E), N, bias=b, out=out)
    ((want, terms),), e = _products([w], x, ids, N)
    live = ((ids >= 0) & (ids < E)).cuda()
    assert (got[~live] == 77).all()
    be = b.double()[e]
    _check(got[live], (want + be)[live], terms[live], K, be[live])


@pytest.mark.parametrize("T,k,E,N,K", [(1, 8, 32, 768, 2048), (2, 2, 4, 40, 96), (200, 4, 6, 300, 512), (900, 2, 4, 128, 288)])
def test_swiglu(T, k, E, N, K, route):
    (G, g), (U, u) = _weights(N, K, 11, count=E), _weights(N, K, 12, count=E)
    ids = _ids(T, k, E, 13)
    x = _randn((T, K), F16, 14)
    got = ops.moe_mx4_swiglu(G, U, x, ops.moe_plan(ids.cuda(), E), N, out_dtype=F32)
    ((a, sa), (b, sb)), _ = _products([g, u], x, ids, N)
    want = torch.nn.functional.silu(a) * b
    # |d silu| <= 1.1 |d gate|; silu itself: exp within 2 units, a sum and a quotient: 2^-21
    ea, eb = (K + 64) * 2.0 ** -24 * sa, (K + 64) * 2.0 ** -24 * sb
    bound = 1.1 * ea * (b.abs() + eb) + torch.nn.functional.silu(a).abs() * eb + want.abs() * 2.0 ** -20
    assert ((got.double() - want).abs() <= bound + 1e-30).all()


def test_swiglu_of_large_gates():
    """silu(-large) is a zero, not a NaN."""
    T, k, E, N, K = 2, 1, 1, 64, 256
    b = ref.random_blocks(N * K // 32, 4, lo=180, hi=181).cuda()
    G = ops.mx4_pack(b.reshape(-1), N, K)
    U, _ = _weights(N, K, 5)
    x = _randn((T, K), F32, 6)
    plan = ops.moe_plan(torch.zeros(T, k, dtype=torch.int32).cuda(), E)
    got = ops.moe_mx4_swiglu(G, U, x, plan, N)
    gate = ops.moe_mx4_linear(G, x, plan, N)
    assert torch.isfinite(got).all() and (got[gate < -200] == 0).all() and (gate < -200).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (1, 8, 2048), (7, 3, 77), (130, 6, 1000), (3, 32, 512)])
def test_combine(T, k, N, dtype):
    y, w = _randn((T, k, N), dtype, 1), torch.rand(T, k, device="cuda") - 0.3
    ids = _ids(T, k, 40, 2, drop=0.2).cuda()
    ids[0, 0] = -1
    y[ids < 0] = NAN  # rows that no product has written
    z = torch.where((ids >= 0)[:, :, None], y.double(), 0.0) * w.double()[:, :, None]
    want = z.sum(1)
    got = ops.moe_combine(y, ids, w)
    eps = torch.finfo(dtype).eps / 2
    bound = z.abs().sum(1) * (k * 2.0 ** -24) * 1.01 + want.abs() * eps * 1.01 + torch.finfo(dtype).smallest_normal * eps
    assert got.dtype == dtype and ((got.double() - want).abs() <= bound).all()
    assert (ops.moe_combine(y, torch.full_like(ids, -1), w) == 0).all()
    few = ops.moe_combine(y, ids, w, experts=20)
    assert torch.equal(few, ops.moe_combine(y, torch.where(ids < 20, ids, -1), w))


def _layer(logits, x, G, U, D, k, N, K):
    ids, weights, plan = ops.moe_route(logits, k)
    h = ops.moe_mx4_swiglu(G, U, x, plan, N, out_dtype=x.dtype)
    y = ops.moe_mx4_linear(D, h, plan, K, out_dtype=x.dtype)
    return ids, weights, h, y, ops.moe_combine(y, ids, weights, experts=logits.shape[1])


@pytest.mark.parametrize("T", [1, 37, 300])
def test_a_layer(T):
    """Router to sum, as a model runs it, and the same captured once and replayed with other tokens and other routes."""
    k, E, N, K = 4, 16, 384, 512
    (G, g), (U, u), (D, d) = _weights(N, K, 1, E), _weights(N, K, 2, E), _weights(K, N, 3, E)

    def inputs(seed):
        return _randn((T, E), F32, seed), _randn((T, K), BF16, seed + 1)

    logits, x = inputs(20)
    ids, weights, h, y, out = _layer(logits, x, G, U, D, k, N, K)
    ((a, _), (b, _)), _ = _products([g, u], x, ids.cpu(), N)
    assert ((h.double() - torch.nn.functional.silu(a) * b).norm() / h.double().norm()).item() < 2.0 ** -8
    ((want, terms),), _ = _products([d], h, ids.cpu(), K)
    _check(y, want, terms, N)
    assert ((out.double() - torch.einsum("tkn,tk->tn", y.double(), weights.double())).norm() / out.double().norm()).item() < 2.0 ** -8
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _layer(logits, x, G, U, D, k, N, K)
    for seed in (20, 30, 40):
        a, b = inputs(seed)
        logits.copy_(a)
        x.copy_(b)
        if seed == 40:
            logits[T // 2:, 3:] = -INF  # fewer experts than k: pairs without one
        graph.replay()
        fresh = _layer(logits, x, G, U, D, k, N, K)
        live = fresh[0] >= 0
        for got, want in zip(captured, fresh):
            assert torch.equal(got[live], want[live]) if got.dim() == 3 else torch.equal(got, want)
    assert ops.device_status() == 0
