"""The largest number of rows that the microscaled 4-bit linear product takes:
2^28 - 16 rows of one channel, whose pieces fill a launch, so that the scales'
planes take another.  Against oracle/mxfp4.py in 64 bits."""
import pytest
import torch

from oracle import mxfp4 as O
from test_gpu_mxfp4 import assert_within, dev, say, weight

pytestmark = pytest.mark.gpu


def test_most_rows():
    from spider_moe_amd import ForgeGEMM
    n, k, n_out = (1 << 28) - 16, 1, 3
    say("most rows")
    x = torch.randn(n, k, device=dev, generator=torch.Generator(device=dev).manual_seed(1), dtype=torch.bfloat16)
    codes, scale = weight(n_out, k)
    got = ForgeGEMM().linear_mxfp4(x, codes, scale)
    for at in (slice(0, 3000), slice((1 << 27) - 1000, (1 << 27) + 1000), slice(n - 3000, n)):
        want, err = O.linear(x[at], codes, scale)
        assert_within(got[at], want, err)
    del got
    torch.cuda.empty_cache()
    with pytest.raises(RuntimeError):
        ForgeGEMM().linear_mxfp4(torch.zeros(n + 1, 1, dtype=torch.bfloat16, device=dev), codes, scale)


@pytest.mark.parametrize("n", [1, 20, 60])
def test_codes_far_apart(n):
    """Codes and scales as columns of tables whose rows lie more than 2^22 bytes
    apart."""
    from spider_moe_amd import ForgeGEMM
    say("far codes", n)
    k, n_out = 200, 40
    codes, scale = weight(n_out, k)
    x = torch.randn(n, k, generator=torch.Generator().manual_seed(n)).bfloat16().to(dev)
    want = ForgeGEMM().linear_mxfp4(x, codes, scale)
    table = torch.zeros(n_out, (1 << 22) + 4096, dtype=torch.uint8, device=dev)
    far, fars = table[:, 16:16 + codes.shape[1]], table[:, 1024:1024 + scale.shape[1]]
    far.copy_(codes)
    fars.copy_(scale)
    assert torch.equal(ForgeGEMM().linear_mxfp4(x, far, fars), want)
