"""MXFP4 products on the B200 where FP32 holds every sum exactly (mx4_exact.py): the results have to be the 64-bit ones, bit for bit, in each kernel, whatever the
length of the columns. A stage left out, a remainder dropped, a stale scale or a single element off by one code shows here."""
import pytest

torch = pytest.importorskip("torch")
import mx4_exact as exact
import mx4_reference as ref
from test_gpu_moe import _ids, _products
from test_gpu_mx4 import BF16, F16, F32, _randn, _weights, route  # noqa: F401

from brotensor_b200 import ops

pytestmark = pytest.mark.gpu


def _case(M, N, K, dtype=BF16, seed=1):
    b = exact.weights(N, K, seed).cuda()
    x = exact.activations((M, K), dtype, seed + 1, device="cuda")
    w = ref.matrix(b, N, K)
    assert exact.sums_are_exact(x.double(), w)
    return ops.mx4_pack(b.reshape(-1), N, K), x, x.double() @ w.T


@pytest.mark.parametrize("M", [1, 2, 8, 16, 17, 45, 100, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 32), (77, 96), (130, 2304 + 32), (1024, 4096), (700, 7168)])
def test_linear(M, N, K, route):
    W, x, want = _case(M, N, K)
    exact.same(ops.mx4_linear(W, x, N, out_dtype=F32), want)


@pytest.mark.parametrize("K", [14336, 65536, 65536 + 32, 131072])
@pytest.mark.parametrize("M", [1, 2, 16, 40, 200])
def test_long_columns(M, K, route):
    W, x, want = _case(M, 130, K)
    exact.same(ops.mx4_linear(W, x, 130, out_dtype=F32), want)


@pytest.mark.parametrize("M,N,K", [(40, 4608, 4096), (72, 4608, 2048), (65, 4300, 1056), (72, 2048, 8192), (87, 1700, 8224), (100, 512, 6176), (119, 1000, 6400), (119, 4224, 6144), (513, 640, 4096)])
def test_rows_between_the_two_forms(M, N, K, route):
    W, x, want = _case(M, N, K)
    exact.same(ops.mx4_linear(W, x, N, out_dtype=F32), want)


@pytest.mark.parametrize("M,N,K", [(1, 14336, 4096), (8, 1024, 14336), (16, 2048, 4096), (40, 1024, 4096)])
def test_split_sums_again_and_again(M, N, K):
    """K cut over the CTAs of clusters, whose sums cross from SM to SM: the same bits on every one of many calls, with other launches between."""
    W, x, want = _case(M, N, K)
    want = want.float()
    out = torch.empty(M, N, device="cuda")
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(400):
        out.fill_(float(turn))
        ops.mx4_linear(W, x, N, out=out)
        wrong += (out != want).sum()
    if wrong.item():
        exact.same(out, want.double())
    assert wrong.item() == 0, f"{wrong.item()} results differed in one of the calls"
    assert ops.device_status() == 0


@pytest.mark.parametrize("per_pair", [False, True])
@pytest.mark.parametrize("T,k,E,N,K", [(1, 8, 128, 256, 512), (3, 2, 8, 77, 96), (50, 4, 16, 200, 544), (300, 2, 3, 130, 256), (96, 6, 64, 384, 1408), (700, 4, 5, 128, 320)])
def test_experts(T, k, E, N, K, per_pair, route):
    b = exact.weights(N, K, 1, count=E).cuda()
    w = ref.matrix(b, E * N, K).reshape(E, N, K)
    ids = _ids(T, k, E, T)
    x = exact.activations((T, k, K) if per_pair else (T, K), F16, 3, device="cuda")
    ((want, terms),), _ = _products([w], x, ids, N)
    assert terms.max() < 2 ** 22
    got = ops.moe_mx4_linear(ops.mx4_pack(b.reshape(-1), N, K, count=E), x, ops.moe_plan(ids.cuda(), E), N, out_dtype=F32)
    exact.same(got.reshape(T * k, N), want.reshape(T * k, N))


# Gated: 16 experts of up to 496 rows and 113 to 140 pairs leave little shared memory beside the partial sums.
@pytest.mark.parametrize("T,k,E,N,K", [(1, 8, 32, 384, 1024), (20, 7, 16, 496, 3200), (57, 2, 16, 130, 2048), (200, 4, 6, 300, 512)])
def test_both_products_of_a_gated_one(T, k, E, N, K, route):
    """gate = up: the result depends on one product alone, which is exact, so that silu(g) g is off by silu's own error: exp within 2^-22 of its value or |g| 2^-24 of it,
    a sum, a quotient within 2^-22 and a product."""
    b = exact.weights(N, K, 1, count=E).cuda()
    w = ref.matrix(b, E * N, K).reshape(E, N, K)
    W = ops.mx4_pack(b.reshape(-1), N, K, count=E)
    ids = _ids(T, k, E, T)
    x = exact.activations((T, K), BF16, 3, device="cuda")
    ((g, terms),), _ = _products([w], x, ids, N)
    assert terms.max() < 2 ** 22
    got = ops.moe_mx4_swiglu(W, W, x, ops.moe_plan(ids.cuda(), E), N, out_dtype=F32).double()
    want = torch.nn.functional.silu(g) * g
    bound = want.abs() * (2.0 ** -20 + (-g).clamp(min=0) * 2.0 ** -23) + 2.0 ** -126 * g.abs() ** 2
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (8, 1024, 14336), (45, 2560, 6912), (2, 130, 131072), (513, 640, 4096)])
def test_the_norm_of_inexact_sums(M, N, K, route):
    """Sums that FP32 does not hold: each of the K / 64 steps rounds the accumulator once, by 2^-23 of it at most, one way or the other."""
    W, w = _weights(N, K, 17)
    x = _randn((M, K), BF16, 18)
    want = ref.quantise(x) @ w[0].T
    got = ops.mx4_linear(W, x, N, out_dtype=F32).double()
    assert ((got - want).norm() / want.norm()).item() < (K / 64) ** 0.5 * 2.0 ** -23
