"""Which layout of scales a microscaled 4-bit linear product takes (CPU, by the
workspace query): planes of both operands' scales for the large tiles, the
user's rows for everything else.  A few rows never run on large tiles, however
many channels there are."""
import pytest


@pytest.fixture(scope="module")
def need():
    from spider_moe_amd import _native
    return _native.lib().smoe_linear_mxfp4_workspace_bytes


def rows_only(n, k):
    """Bytes of the quantized rows alone, each buffer a multiple of 256."""
    blocks = -(-k // 32)
    up = lambda b: (b + 255) // 256 * 256
    return up(n * 16 * blocks) + up((n + 3) // 4 * 16 * -(-blocks // 4))


@pytest.mark.parametrize("n_out", [40704, 40705, 50257, 65536, 1 << 22])
@pytest.mark.parametrize("n,k", [(1, 32768), (2, 16384), (8, 4096), (9, 2048), (16, 2816), (17, 32), (24, 1024)])
def test_few_rows_take_no_planes(need, n, k, n_out):
    assert need(n, k, n_out) == rows_only(n, k)


@pytest.mark.parametrize("n,n_out", [(25, 40705), (100, 50257), (2000, 5000), (2500, 4096)])
def test_large_products_take_planes(need, n, n_out):
    k = 257
    planes = (n_out + 3) // 4 * 16 * 3  # nine blocks are three words
    assert need(n, k, n_out) == rows_only(n, k) + (planes + 255) // 256 * 256


@pytest.mark.parametrize("n,n_out", [(25, 40704), (256, 40704), (257, 20224)])
def test_products_below_take_none(need, n, n_out):
    assert need(n, 257, n_out) == rows_only(n, 257)


def test_rows_further_apart_than_the_product_takes_are_copied():
    """Codes as columns of a table whose rows lie more than 2^22 bytes apart."""
    import torch
    from spider_moe_amd.quant import _pitched
    table = torch.zeros(3, (1 << 22) + 16, dtype=torch.uint8)
    table[:, :48] = torch.arange(3 * 48).view(3, 48)
    far = table[:, :48]
    t, ld = _pitched(far, 48, 16, most=1 << 22)
    assert ld == 48 and t.data_ptr() != far.data_ptr() and torch.equal(t, far)
    assert _pitched(far, 48, 16)[0] is far and _pitched(far[:1], 48, 16, most=1 << 22)[0].data_ptr() == far.data_ptr()
