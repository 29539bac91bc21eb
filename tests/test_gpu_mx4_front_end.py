"""What the Python front end of the MXFP4 and expert operators refuses on a machine with a GPU: the check that says what is wrong is reached."""
import pytest

torch = pytest.importorskip("torch")
from brotensor_b200 import ops

pytestmark = pytest.mark.gpu


def _image(n, k, count=1):
    return torch.zeros(count * ops.mx4_image_bytes(n, k), dtype=torch.uint8, device="cuda")


def test_refusals():
    c = dict(device="cuda")
    x, W = torch.ones(4, 64, **c), _image(40, 64)
    for call, why in (
            (lambda: ops.mx4_linear(W.cpu(), x, 40), "an image is"),
            (lambda: ops.mx4_linear(W, x.cpu(), 40), "X is on"),
            (lambda: ops.mx4_linear(W[1:], x, 40), "the image holds"),
            (lambda: ops.mx4_linear(W, x, 400), "the image holds"),
            (lambda: ops.mx4_linear(W, x.int(), 40), "X must be"),
            (lambda: ops.mx4_linear(W, torch.ones(64, 4, **c).t(), 40), "X must be"),
            (lambda: ops.mx4_linear(W, torch.ones(4, 48, **c), 40), "multiple of 32"),
            (lambda: ops.mx4_linear(W, x, 40, bias=torch.ones(40, dtype=torch.float16, **c)), "bias must have"),
            (lambda: ops.mx4_linear(W, x, 40, bias=torch.ones(39, **c)), "bias must have"),
            (lambda: ops.mx4_linear(W, x, 40, out=torch.empty(4, 41, **c)), "out must be"),
            (lambda: ops.mx4_linear(W, x, 40, out=torch.empty(4, 40, **c), out_dtype=torch.float16), "out must be"),
            (lambda: ops.mx4_linear(W, torch.ones(30, 64, **c), 40, ws=torch.empty(100000, **c)), "ws must be"),
            (lambda: ops.mx4_linear(W, torch.ones(30, 64, **c), 40, ws=torch.empty(100, dtype=torch.uint8, **c)), "workspace"),
            (lambda: ops.mx4_quantize(x.int()), "x must be"), (lambda: ops.mx4_quantize(x[0]), "x must be"),
            (lambda: ops.mx4_quantize(x, out=W[1:]), "the image holds"),
            (lambda: ops.mx4_dequantize(W, 40, 64, out_dtype=torch.int32), "out_dtype"),
            (lambda: ops.mx4_dequantize(W, 400, 64), "the image holds"),
            (lambda: ops.mx4_gemm(W, ops.mx4_quantize(x), 4, 40, 64, bias=torch.ones(3, **c)), "bias must have"),
            (lambda: ops.moe_route(x.int(), 2), "logits must be"), (lambda: ops.moe_route(x, 65), "supported sizes"),
            (lambda: ops.moe_route(torch.ones(4, 8, **c), 9), "more than E"), (lambda: ops.moe_route(torch.ones(4, 2000, **c), 2), "supported sizes"),
            (lambda: ops.moe_plan(torch.zeros(4, 2, **c), 8), "ids must be"),
            (lambda: ops.moe_plan(torch.zeros(2, 4, dtype=torch.int32, **c).t(), 8), "ids must be"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=why):
            call()
    plan, E3 = ops.moe_plan(torch.zeros(4, 2, dtype=torch.int32, **c), 3), _image(40, 64, 3)
    for call, why in (
            (lambda: ops.moe_mx4_linear(W, x, plan, 40), "the image holds"),
            (lambda: ops.moe_mx4_linear(E3, x[:3], plan, 40), "as the plan"),
            (lambda: ops.moe_mx4_linear(E3, torch.ones(4, 3, 64, **c), plan, 40), "as the plan"),
            (lambda: ops.moe_mx4_linear(E3, x.half().int(), plan, 40), "X must be"),
            (lambda: ops.moe_mx4_linear(E3, x.cpu(), plan, 40), "X is on"),
            (lambda: ops.moe_mx4_linear(E3, x, plan, 40, bias=torch.ones(40, **c)), "bias must be"),
            (lambda: ops.moe_mx4_swiglu(E3, W, x, plan, 40), "the image holds"),
            (lambda: ops.moe_mx4_linear(E3, x, plan, 40, out=torch.empty(4, 40, **c)), "out must be"),
            (lambda: ops.moe_combine(x, torch.zeros(4, 2, dtype=torch.int32, **c), torch.ones(4, 2, **c)), "y must be"),
            (lambda: ops.moe_combine(torch.ones(4, 2, 8, **c), torch.zeros(4, 2, **c), torch.ones(4, 2, **c)), "ids must be"),
            (lambda: ops.moe_combine(torch.ones(4, 2, 8, **c), torch.zeros(4, 2, dtype=torch.int32, **c), torch.ones(4, 3, **c)), "weights must be"),
            (lambda: ops.moe_combine(torch.ones(4, 2, 8, **c).int(), torch.zeros(4, 2, dtype=torch.int32, **c), torch.ones(4, 2, **c)), "y must be"),
    ):
        with pytest.raises((ValueError, RuntimeError), match=why):
            call()
    assert ops.moe_mx4_linear(E3, x, plan, 40).shape == (4, 2, 40) and ops.device_status() == 0
