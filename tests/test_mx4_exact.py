"""The exact products of mx4_exact.py can tell: a wrong element, a missing block, a stale scale all show. (On the CPU.)"""
import pytest

torch = pytest.importorskip("torch")
import mx4_exact as exact
import mx4_reference as ref


@pytest.fixture(scope="module", params=[256, 14336, 131072])
def case(request):
    K = request.param
    b = exact.weights(3, K, 1)
    return K, b, ref.matrix(b, 3, K), exact.activations((2, K), torch.float32, 2)


def test_the_activations_stay_as_they_are(case):
    K, _, w, x = case
    assert torch.equal(ref.quantise(x), x.double()) and torch.equal(x.half().float(), x) and torch.equal(x.bfloat16().float(), x)
    assert exact.sums_are_exact(x.double(), w)


def test_fp32_sums_are_exact_in_any_order(case):
    K, _, w, x = case
    want = x.double() @ w.T
    p = torch.randperm(K, generator=torch.Generator().manual_seed(3))
    terms = x[:, None, p] * w.float()[None][:, :, p]
    assert torch.equal(terms.double(), x.double()[:, None, p] * w[None][:, :, p])
    assert torch.equal(terms.sum(-1).double(), want)
    acc = torch.zeros(2, 3)
    for c in terms.unflatten(-1, (-1, 64)).sum(-1).unbind(-1):
        acc += c
    exact.same(acc, want)


@pytest.mark.parametrize("what", ["one code", "a block of 32", "a tile of 256", "a scale", "one activation"])
def test_a_mistake_shows(case, what):
    K, b, w, x = case
    want = x.double() @ w.T
    q, bad = x.double().clone(), b.reshape(3, K // 32, 17).clone()
    at = K // 32 - 1
    if what == "one code":
        bad[1, at, 9] ^= 1
    elif what == "a block of 32":
        bad[1, at, 1:] = 0
    elif what == "a tile of 256":
        q[:, -256:] = 0
    elif what == "a scale":
        bad[2, at, 0] += 1
    else:
        q[1, K - 1] += 0.5
    with pytest.raises(AssertionError, match="differ"):
        exact.same((q @ ref.matrix(bad, 3, K).T).float(), want)
