"""Sizes at the edge of what a launch takes (2^32 threads) are refused up
front: no call below gets as far as a launch."""
import pytest

FAKE = 0x1000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    from spider_moe_amd import _native
    return _native.lib()


@pytest.mark.parametrize("n", [(1 << 26) - 3, (1 << 26) - 2, (1 << 26) - 1, 1 << 26, (1 << 31) - 1])
def test_select_groups_rows(lib, n):
    from spider_moe_amd import _native as nat
    assert lib.smoe_select_groups(FAKE, nat.F32, n, 4, 2, 1, None, 1, 1, 1, 1.0, FAKE, FAKE, None) == 1
    assert "2^26" in lib.smoe_last_error().decode()
    assert lib.smoe_select_groups_backward(FAKE, nat.F32, n, 4, 2, 1, 1, 1.0, FAKE, FAKE, FAKE, None) == 1
    assert "2^26" in lib.smoe_last_error().decode()


@pytest.mark.parametrize("g,rows,cols,block_rows", [
    (1, (1 << 28) - 15, 128, 1), (1, (1 << 28) - 1, 128, 1), (1, 1 << 28, 128, 1), (1, (1 << 27) - 7, 256, 1),
    (3, 89478481, 128, 1), (1, (1 << 24) * 128 - 127, 128, 128), (1 << 24, 1, 128, 128)])
def test_quantizer_blocks(lib, g, rows, cols, block_rows):
    from spider_moe_amd import _native as nat
    assert lib.smoe_quantize_fp8_blocks(FAKE, nat.F32, g, rows, cols, cols, block_rows, FAKE, cols, FAKE, None) == 1
    assert "blocks of" in lib.smoe_last_error().decode()
