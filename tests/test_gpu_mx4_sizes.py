"""Sizes at the end of an int, where memory allows them."""
import pytest

torch = pytest.importorskip("torch")
from brotensor_b200 import ops

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def test_the_longest_rows_of_a_sum():
    """2^31 - 1 columns, an odd number: one at a time, and as many threads as an int counts."""
    N = 2 ** 31 - 1
    y = torch.zeros(1, 1, N, dtype=F16, device="cuda")
    for i in (0, 1, 255, 2 ** 30 + 7, N - 1):
        y[0, 0, i] = i % 13 + 1
    out = torch.empty(1, N, dtype=F16, device="cuda")
    out[0, -5000:] = 7
    ops.moe_combine(y, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1, 1), 0.5, device="cuda"), out=out)
    for i in (0, 1, 255, 2 ** 30 + 7, N - 1):
        assert out[0, i].item() == (i % 13 + 1) / 2
    assert out[0, -5000:].count_nonzero().item() == 1


def test_rows_that_a_c_int_does_not_hold():
    """2^32 + 32 columns: their low 32 bits are a legal 32."""
    x = torch.empty(1, 2 ** 32 + 32, dtype=F16, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.mx4_quantize(x)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.mx4_linear(torch.empty(17408, dtype=torch.uint8, device="cuda"), x, 4)
    with pytest.raises(ValueError, match="supported sizes"):
        ops.moe_route(x, 2)
