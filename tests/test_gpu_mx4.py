"""MXFP4 images and their products on the B200, against the definitions in 64 bits.

Tolerances. Quantisation and decoding are exact. A product is a sum of K exact terms a b in FP32: the tensor cores add 64 of them at a
time to the accumulator, each cut to at least 24 bits below the largest term, so a result is at most (K + 64) 2^-24 S off,
S = sum |a b|; the partial sums of a split K add 8 roundings, inside that. Then half a step of the output type."""
import pytest

torch = pytest.importorskip("torch")
import mx4_reference as ref

from brotensor_b200 import ops

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g)
    x[..., ::37] *= 9
    return x.to(dtype)


def _weights(rows, K, seed, count=1):
    b = ref.random_blocks(count * rows * (K // 32), seed).cuda()
    return ops.mx4_pack(b.reshape(-1), rows, K, count=count), ref.matrix(b, count * rows, K).reshape(count, rows, K)


def _check(got, want, terms, K, bias=None):
    """`terms`: sum of |a b| of each result."""
    eps = torch.finfo(got.dtype).eps / 2
    size = want.abs() if bias is None else want.abs() + bias.abs()
    bound = (K + 64) * 2.0 ** -24 * terms + eps * 1.01 * size + 2.0 ** -24 * size + torch.finfo(got.dtype).smallest_normal * eps
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"{int((off > bound).sum())} of {off.numel()} off, the worst {float((off / bound).max()):.3g} times what is allowed"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (7, 256), (129, 288), (300, 1024), (5, 4096)])
def test_quantise_is_exact(rows, K, dtype):
    x = _randn((rows, K), dtype, rows + K)
    x[0, :32] = 0
    image = ops.mx4_quantize(x)
    assert image.numel() == ops.mx4_image_bytes(rows, K)
    assert torch.equal(ops.mx4_dequantize(image, rows, K), ref.quantise(x).float())
    assert torch.equal(ops.mx4_dequantize(image, rows, K, out_dtype=BF16), ref.quantise(x).to(BF16))
    assert torch.equal(ops.mx4_dequantize(image, rows, K, out_dtype=F16), ref.quantise(x).to(F16))


def test_quantise_borders():
    """Every midpoint and its neighbours, at scales from the smallest to the largest."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99])
    m = torch.cat([mids, mids.nextafter(torch.tensor(0.0)), mids.nextafter(torch.tensor(9.0))])
    rows = []
    for e in (-149, -140, -129, -128, -127, -126, -125, -60, 0, 3, 60, 124, 125):
        r = torch.zeros(32)
        r[:30] = m * torch.tensor([1.0, -1.0]).repeat(15)
        r[30] = 4.0
        rows.append(torch.ldexp(r.double(), torch.tensor(e)).float())
    x = torch.stack(rows).cuda()
    assert torch.isfinite(x).all()
    assert torch.equal(ops.mx4_dequantize(ops.mx4_quantize(x), len(rows), 32), ref.quantise(x).float())


def test_quantise_not_finite():
    x = _randn((4, 128), F32, 5)
    x[1, 40], x[2, 3], x[3, 127] = float("inf"), float("nan"), float("-inf")
    got, want = ops.mx4_dequantize(ops.mx4_quantize(x), 4, 128), ref.quantise(x).float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    assert int(got.isnan().sum()) == 96


@pytest.mark.parametrize("rows,K,count", [(1, 32, 1), (130, 96, 1), (128, 256, 3), (65, 320, 5), (256, 4096, 2)])
def test_pack_keeps_every_bit(rows, K, count):
    g = torch.Generator().manual_seed(rows + K)
    b = torch.randint(0, 256, (count * rows * K // 32, 17), generator=g, dtype=torch.uint8)
    image = ops.mx4_pack(b.cuda().reshape(-1), rows, K, count=count)
    size = ops.mx4_image_bytes(rows, K)
    for c in range(count):
        got = ops.mx4_dequantize(image[c * size:(c + 1) * size], rows, K)
        want = ref.matrix(b, count * rows, K).reshape(count, rows, K)[c].float().cuda()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0, 0, 0), want.nan_to_num(0, 0, 0))


def test_pack_takes_blocks_from_any_byte():
    b = ref.random_blocks(64 * 8, 3).cuda()
    shifted = torch.zeros(b.numel() + 5, dtype=torch.uint8, device="cuda")
    shifted[5:] = b.reshape(-1)
    assert torch.equal(ops.mx4_dequantize(ops.mx4_pack(shifted[5:], 64, 256), 64, 256), ref.matrix(b, 64, 256).float())


@pytest.fixture(params=["as routed", "small tiles", "wide tiles", "few rows"])
def route(request):
    """Each kernel takes every call (that of few rows, every call of up to 16 of them) and is held to the definition whatever the routing rules say."""
    was = ops.get_option("mx4_wide"), ops.get_option("mx4_few")
    ops.set_option("mx4_wide", {"small tiles": 0, "wide tiles": 2}.get(request.param, was[0]))
    ops.set_option("mx4_few", {"small tiles": 0, "wide tiles": 0, "few rows": 16}.get(request.param, was[1]))
    yield
    ops.set_option("mx4_wide", was[0])
    ops.set_option("mx4_few", was[1])


@pytest.mark.parametrize("M", [1, 2, 16, 17, 100, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(128, 256), (1, 32), (77, 96), (200, 544), (384, 1024)])
def test_linear(M, N, K, route):
    W, w = _weights(N, K, N + K)
    x = _randn((M, K), F32, M + K)
    q = ref.quantise(x)
    want, terms = q @ w[0].T, q.abs() @ w[0].abs().T
    _check(ops.mx4_linear(W, x, N), want, terms, K)


@pytest.mark.parametrize("x_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("y_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_types(x_dtype, y_dtype, bias, route):
    M, N, K = 21, 150, 416
    W, w = _weights(N, K, 7)
    x = _randn((M, K), x_dtype, 8)
    b = _randn((N,), x_dtype, 9) if bias else None
    q = ref.quantise(x)
    want = q @ w[0].T + (b.double() if bias else 0)
    _check(ops.mx4_linear(W, x, N, bias=b, out_dtype=y_dtype), want, q.abs() @ w[0].abs().T, K, b.double() if bias else None)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (8, 1024, 14336), (45, 2560, 6912), (513, 640, 4096), (1, 128, 65536), (2, 130, 2304 + 32), (2100, 5000, 512)])
def test_linear_long(M, N, K, route):
    W, w = _weights(N, K, 17)
    x = _randn((M, K), BF16, 18)
    q = ref.quantise(x)
    want = q @ w[0].T
    got = ops.mx4_linear(W, x, N, out_dtype=F32)
    _check(got, want, q.abs() @ w[0].abs().T, K)
    assert ((got - want).norm() / want.norm()).item() < 1e-5
    assert torch.equal(got, ops.mx4_linear(W, x, N, out_dtype=F32)), "the same call gives other bits"


def test_linear_nothing_to_do():
    W, _ = _weights(64, 64, 1)
    assert ops.mx4_linear(W, torch.empty(0, 64, device="cuda"), 64).shape == (0, 64)
    assert ops.mx4_quantize(torch.empty(0, 64, device="cuda")).numel() == 0
    assert ops.mx4_linear(torch.empty(0, dtype=torch.uint8, device="cuda"), torch.ones(3, 64, device="cuda"), 0).shape == (3, 0)


def test_linear_not_finite_stays_in_its_row():
    W, w = _weights(300, 512, 2)
    x = _randn((40, 512), F32, 3)
    x[7, 100], x[30, 511] = float("nan"), float("inf")
    got = ops.mx4_linear(W, x, 300)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 30]] = True
    assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()


def test_gemm_of_images_and_outputs_given():
    M, N, K = 70, 200, 768
    W, w = _weights(N, K, 4)
    x = _randn((M, K), F16, 5)
    image = ops.mx4_quantize(x)
    want = ops.mx4_linear(W, x, N, out_dtype=F32)
    assert torch.equal(ops.mx4_gemm(W, image, M, N, K), want)
    guard = torch.full((M + 2, N), 123.0, device="cuda")
    ops.mx4_gemm(W, image, M, N, K, out=guard[1:M + 1])
    assert torch.equal(guard[1:M + 1], want) and (guard[0] == 123).all() and (guard[-1] == 123).all()
    big = torch.empty(ops.mx4_image_bytes(M, K) + 4096, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.mx4_linear(W, x, N, out_dtype=F32, ws=big), want)


def test_linear_on_a_side_stream_and_in_a_graph():
    M, N, K = 5, 512, 2048
    W, w = _weights(N, K, 6)
    x = _randn((M, K), BF16, 7)
    want = ops.mx4_linear(W, x, N)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.mx4_linear(W, x, N)
    side.synchronize()
    assert torch.equal(y, want)
    xs, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = ops.mx4_linear(W, xs, N)
    for seed in (7, 8, 9):
        xs.copy_(_randn((M, K), BF16, seed))
        graph.replay()
        assert torch.equal(ys, ops.mx4_linear(W, xs, N))
    assert ops.device_status() == 0
