"""The quantizer on the pairs where a quotient comes nearest to a wrong
rounding (tests/test_fp8_blocks_quotient.py names them), bit for bit the CPU
formula's codes."""
import pytest
import torch

from test_fp8_blocks_quotient import critical_pairs
from test_gpu_fp8_blocks import dev, same_codes, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block_rows", [1, 128])
def test_codes_of_the_critical_pairs(block_rows):
    from spider_moe_amd import quantize_fp8_blocks
    say("critical quotients", block_rows)
    by_b = {}
    for a, b, _ in critical_pairs():
        by_b.setdefault(float(b), set()).add(float(a))
    rows, scales = [], []
    for b, values in sorted(by_b.items()):
        s = torch.tensor(b)
        amax = next((c for c in (torch.nextafter(448 * s, torch.tensor(0.0)), 448 * s,
                                 torch.nextafter(448 * s, torch.tensor(1e9))) if c / 448 == s), None)
        if amax is None:  # no amax gives this scale
            continue
        a = torch.tensor(sorted(values))
        a = torch.cat([a * 2.0 ** i for i in (-10, -6, 0, 3, 7)])  # subnormal codes to the largest ones
        for part in a.split(127):
            row = torch.zeros(128)
            row[0] = amax
            row[1:1 + part.numel()] = part
            rows.append(torch.where(torch.arange(128) % 3 == 1, -row, row))
            scales.append(b)
    x = torch.stack(rows)
    if block_rows == 128:  # a scale to each block: one row of it, zeros below
        x = torch.nn.functional.pad(x.unsqueeze(1), (0, 0, 0, 2))
    else:
        x = x.unsqueeze(1)
    q, s = quantize_fp8_blocks(x.to(dev), block_rows=block_rows)
    cq, cs = quantize_fp8_blocks(x, block_rows=block_rows)
    assert torch.equal(s.cpu(), cs) and torch.equal(cs.amax(dim=(1, 2)), torch.tensor(scales))
    assert len(set(scales)) > 100
    assert same_codes(q, cq)
