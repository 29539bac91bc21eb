"""Sizes that no call takes have no size either, and none of them is folded into one that would be taken. (Without a device.)"""
import pytest

torch = pytest.importorskip("torch")
from brotensor_b200 import _capi as capi
from brotensor_b200 import ops

MOST = 2 ** 31 - 1 - 1024 * 128  # pairs


@pytest.mark.parametrize("tokens,k", [(MOST + 1, 1), (MOST // 32 + 1, 32), (2 ** 40, 2), (2 ** 62, 4), (2 ** 63 - 1, 32), (2 ** 59, 32)])
def test_sizes_of_more_pairs_than_a_plan_holds_are_0(tokens, k):
    L = capi.lib()
    buf = 1 << 20  # (an aligned address that nothing reads)
    assert L.b200q_moe_plan(buf, tokens, k, 64, buf, None) == capi.ERR_UNSUPPORTED
    assert L.b200q_moe_plan_bytes(tokens, k, 64) == 0
    assert L.b200q_moe_mx4_workspace_bytes(tokens, k, 64, 256) == 0
    with pytest.raises(ValueError, match="supported sizes"):
        ops.MoePlan(tokens, k, 64, "meta")


@pytest.mark.parametrize("k", [1, 32])
def test_the_most_pairs_have_a_size(k):
    L = capi.lib()
    assert L.b200q_moe_plan_bytes(MOST // k, k, 1024) > 8 * (MOST // k) * k
    assert L.b200q_moe_mx4_workspace_bytes(MOST // k, k, 1024, 256) >= (MOST // k * k // 128) * 17408


@pytest.mark.parametrize("count,rows", [(2 ** 32, 2 ** 32 + 1), (2 ** 62, 4), (2 ** 63 - 1, 3), (1, 2 ** 34), (2 ** 34, 1)])
def test_pack_of_more_rows_than_64_bits_count(count, rows):
    buf = 1 << 20
    L = capi.lib()
    assert L.b200q_mx4_pack(buf, count, rows, 32, buf, None) == capi.ERR_UNSUPPORTED and b"more than one launch" in L.b200q_last_error()


@pytest.mark.parametrize("experts", [0, -1, -2 ** 31 - 1, -2 ** 32 + 4])
def test_sum_over_no_experts(experts):
    """ctypes would pass the low 32 bits on: -2^32 + 4 are 4 experts."""
    with pytest.raises(ValueError, match="experts"):
        ops.moe_combine(torch.empty(1, 2, 8, device="meta"), torch.empty(1, 2, dtype=torch.int32, device="meta"), torch.empty(1, 2, device="meta"), experts)
