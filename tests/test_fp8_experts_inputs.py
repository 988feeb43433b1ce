"""What sparse_expert_delta_fp8_blocks does with its inputs before a launch:
the expert ids' types."""
import pytest
import torch

NARROW = (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64)


@pytest.mark.parametrize("dtype", NARROW)
@pytest.mark.parametrize("e", [6, 128, 200, 256])
def test_ids_of_every_integer_type(dtype, e):
    """An id keeps its expert whatever integer type holds it, and one outside
    [0, E) stays outside: the type's own limits are no ids of another."""
    from spider_moe_amd.sparse_experts import _expert_ids
    info = torch.iinfo(dtype)
    want = [i for i in (0, 1, 5, 127, 128, 200, 255, 256, 257, -1, -128, 1 << 31, 1 << 32, -(1 << 32), (1 << 63) - 1)
            if info.min <= i <= info.max]
    got = _expert_ids(torch.tensor(want, dtype=dtype), e)
    assert got.dtype == torch.int32
    for w, i in zip(want, got.tolist()):
        assert i == w if 0 <= w < e else not 0 <= i < e, (w, i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_numbers_in_floating_types(dtype):
    from spider_moe_amd.sparse_experts import _expert_ids
    got = _expert_ids(torch.tensor([0, 3, 5, 6, -1, 2.0 ** 33, -(2.0 ** 33)]).to(dtype), 6)
    assert got.tolist() == [0, 3, 5, 6, -1, 6, -1]
