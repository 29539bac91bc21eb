"""MXFP4 products and expert layers where a kernel can go wrong beside its arithmetic: extreme scales, offsets beyond 32 bits, several streams at
once, launches with and without overlap, weights and plans written by the launch just before."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
import mx4_reference as ref
from test_gpu_moe import _ids, _layer, _products
from test_gpu_mx4 import BF16, F16, F32, _check, _randn, _weights, route  # noqa: F401

from brotensor_b200 import ops, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w_e,x_e", [(0, 100), (3, 90), (250, -110), (200, -60), (20, 0)])
def test_extreme_scales(w_e, x_e, route):
    """Scales from 2^-127 up: the sum of the two exponents is what counts."""
    M, N, K = 9, 70, 160
    b = ref.random_blocks(N * K // 32, 3, lo=w_e, hi=w_e + 4).cuda()
    W, w = ops.mx4_pack(b.reshape(-1), N, K), ref.matrix(b, N, K)
    x = (_randn((M, K), F32, 4).double() * 2.0 ** x_e).float()
    q = ref.quantise(x)
    _check(ops.mx4_linear(W, x, N), q @ w.T, q.abs() @ w.abs().T, K)


def test_a_block_of_weights_that_is_not_a_number(route):
    M, N, K = 40, 130, 512
    b = ref.random_blocks(N * K // 32, 3)
    b[5 * K // 32 + 3, 0] = 255
    y = ops.mx4_linear(ops.mx4_pack(b.cuda().reshape(-1), N, K), _randn((M, K), BF16, 4), N)
    assert y[:, 5].isnan().all() and torch.isfinite(torch.cat([y[:, :5], y[:, 6:]], 1)).all()


def test_weights_beyond_four_gigabytes():
    """The last experts of a layer of 64 x 8192 x 16384 (4.6 GB) against the same matrices on their own."""
    E, N, K, k = 64, 8192, 16384, 2
    size = ops.mx4_image_bytes(N, K)
    W = torch.empty(E * size, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for e in (0, 30, 61, 62, 63):
        b = torch.randint(0, 256, (N * K // 32, 17), generator=g, dtype=torch.uint8, device="cuda")
        b[:, 0] = 118
        ops.mx4_pack(b.reshape(-1), N, K, out=W[e * size:(e + 1) * size])
    for T in (2, 20, 800):
        ids = torch.randint(0, 5, (T, k), generator=g, device="cuda")
        ids = torch.tensor([0, 30, 61, 62, 63], device="cuda")[ids].int()
        x = _randn((T, K), BF16, 2)
        y = ops.moe_mx4_linear(W, x, ops.moe_plan(ids, E), N, out_dtype=F32)
        for t in (0, T // 2, T - 1):
            for j in range(k):
                e = int(ids[t, j])
                want = ops.mx4_linear(W[e * size:(e + 1) * size], x[t:t + 1], N, out_dtype=F32)[0]
                assert ((y[t, j] - want).norm() / want.norm()).item() < 1e-6
    assert ops.device_status() == 0


def test_results_beyond_two_to_the_31():
    M, N, K = 140001, 16384, 96
    W, _ = _weights(N, K, 5)
    x = _randn((M, K), BF16, 6)
    y = ops.mx4_linear(W, x, N, out_dtype=BF16)
    assert y.numel() > 2 ** 31
    for lo in (0, 70000, 131070, M - 40):
        assert torch.equal(y[lo:lo + 40], ops.mx4_linear(W, x[lo:lo + 40].contiguous(), N, out_dtype=BF16))
    del y
    image = ops.mx4_quantize(x)
    assert torch.equal(ops.mx4_dequantize(image, M, K, out_dtype=BF16)[-40:], ref.quantise(x[-40:]).to(BF16))


@pytest.mark.parametrize("pdl", [-1, 0, 1])
def test_launches_with_and_without_overlap(pdl):
    """Weights packed, tokens routed and activations written by the launches just before, again and again in the same buffers."""
    T, k, E, N, K = 24, 2, 8, 256, 512
    blocks = [ref.random_blocks(E * N * K // 32, s).cuda().reshape(-1) for s in (1, 2)]
    W = [_weights(N, K, s, E)[1] for s in (1, 2)]
    image = torch.empty(E * ops.mx4_image_bytes(N, K), dtype=torch.uint8, device="cuda")
    logits = [_randn((T, E), F32, s) for s in (3, 4)]
    xs = [_randn((T, K), BF16, s) for s in (5, 6)]
    dense = [ref.quantise(xs[i]) @ W[i][0].T for i in (0, 1)]
    want = []
    for i in (0, 1):
        ids = ref.route(logits[i], k, True, 1.0)[0]
        ((y, terms),), _ = _products([W[i]], xs[i], ids, N)
        want.append((y, terms))
    x, lg = torch.empty_like(xs[0]), torch.empty_like(logits[0])
    ops.set_option("pdl", pdl)
    try:
        got = []
        for turn in range(12):
            i = turn & 1
            ops.mx4_pack(blocks[i], N, K, count=E, out=image)
            x.copy_(xs[i])
            lg.copy_(logits[i])
            _, _, plan = ops.moe_route(lg, k)
            got.append((i, ops.moe_mx4_linear(image, x, plan, N, out_dtype=F32)))
            ops.mx4_pack(blocks[i], N, K, count=E, out=image)
            got.append((i, ops.mx4_linear(image[:ops.mx4_image_bytes(N, K)], x[:1 + turn], N, out_dtype=F32)))
        for i, y in got:
            if y.dim() == 3:
                _check(y, want[i][0], want[i][1], K)
            else:
                assert ((y.double() - dense[i][:len(y)]).norm() / dense[i][:len(y)].norm()).item() < 1e-5
    finally:
        ops.set_option("pdl", 0)
    assert ops.device_status() == 0


def test_several_streams_at_once():
    """Every product kernel of the library that holds tensor memory, on four streams, many times: each finds its columns, all results are right."""
    calls = []
    for M, N, K in ((1, 1024, 4096), (12, 4096, 1024), (40, 2048, 2048), (100, 1024, 4096), (700, 2048, 1024)):
        W, _ = _weights(N, K, M)
        x = _randn((M, K), BF16, M + 1)
        calls.append(lambda W=W, x=x, N=N: ops.mx4_linear(W, x, N))
    for T, k, E, N, K in ((1, 8, 32, 384, 1024), (30, 4, 16, 512, 768), (400, 4, 8, 256, 1024)):
        (G, _), (U, _) = _weights(N, K, 1, E), _weights(N, K, 2, E)
        plan, x = ops.moe_plan(_ids(T, k, E, 3).cuda(), E), _randn((T, K), F16, 4)
        calls.append(lambda G=G, U=U, x=x, plan=plan, N=N: ops.moe_mx4_swiglu(G, U, x, plan, N))
    for M in (33, 300):
        Wq = torch.from_numpy(synth.make_blocks(synth.Q4_K, 1024, 2048, seed=M)).cuda()
        x = _randn((M, 2048), F16, M)
        calls.append(lambda Wq=Wq, x=x: ops.gemm(synth.Q4_K, Wq, x, 1024))
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for c in range(len(calls)):
                    n = (c * (i + 1) + turn) % len(calls)
                    got.append((n, calls[n]()))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for n, y in got:
        assert torch.equal(y, want[n]), n


def test_two_graphs_replayed_in_turn():
    """Two captured layers with workspaces and plans of their own on two streams."""
    k, E, N, K = 2, 8, 256, 512
    (G, _), (U, _), (D, _) = _weights(N, K, 1, E), _weights(N, K, 2, E), _weights(K, N, 3, E)
    made = []
    for T in (3, 60):
        logits, x = _randn((T, E), F32, T), _randn((T, K), BF16, T + 1)
        want = _layer(logits, x, G, U, D, k, N, K)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            got = _layer(logits, x, G, U, D, k, N, K)
        made.append((graph, stream, got, want, logits, x))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _, _ in made:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert ops.device_status() == 0


def test_long_columns_of_few_rows():
    """Rows too long to be quantised inside the launch, and the longest that are."""
    for K in (65536, 65536 + 32, 131072):
        W, w = _weights(130, K, 7)
        x = _randn((2, K), BF16, 8)
        q = ref.quantise(x)
        _check(ops.mx4_linear(W, x, 130, out_dtype=F32), q @ w[0].T, q.abs() @ w[0].abs().T, K)


@pytest.mark.parametrize("M,N,K", [(72, 4608, 2048), (65, 4300, 1056), (72, 2048, 8192), (87, 1700, 8224), (100, 512, 6176), (119, 1000, 6400), (119, 4224, 6144)])
def test_rows_between_the_two_forms(M, N, K):
    """Rows of a size where both forms of the product, and splits of different widths, meet: one CTA an SM, whose clusters do not fill them all."""
    W, w = _weights(N, K, M)
    x = _randn((M, K), BF16, N)
    q = ref.quantise(x)
    _check(ops.mx4_linear(W, x, N, out_dtype=F32), q @ w[0].T, q.abs() @ w[0].abs().T, K)


def test_first_calls_of_a_process_are_captured():
    """What the library asks the device once (attributes, how many clusters it holds) may be asked while a stream is captured."""
    code = """
import torch, mx4_reference as ref
from brotensor_b200 import ops
N, K = 2048, 8192
W = ops.mx4_pack(ref.random_blocks(N * (K // 32), 1).cuda().reshape(-1), N, K)
xs = [torch.randn(M, K, device="cuda") for M in (1, 40, 72, 300)]
ids = torch.randint(0, 4, (50, 2), dtype=torch.int32, device="cuda")
E = ops.mx4_pack(ref.random_blocks(4 * 96 * 8, 2).cuda().reshape(-1), 96, 256, count=4)
def run():
    plan = ops.moe_plan(ids, 4)
    return [ops.mx4_linear(W, x, N) for x in xs] + [ops.moe_mx4_linear(E, xs[0][:, :256].expand(50, 256).contiguous(), plan, 96)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ys = run()
g.replay()
g.replay()
for a, b in zip(ys, run()):
    assert torch.equal(a, b)
assert ops.device_status() == 0
print("same")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here] + os.environ.get("PYTHONPATH", "").split(os.pathsep)))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]
