"""The largest sizes that the microscaled 4-bit entry points take, and the first
ones that they refuse (CPU: refused before any launch)."""
import ctypes

import pytest

FAKE = 0x1000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    from spider_moe_amd import _native
    return _native.lib()


@pytest.mark.parametrize("bad", [dict(k=(1 << 23) + 1, ldx=1 << 24, ldw=1 << 22), dict(no=(1 << 22) + 1),
                                 dict(ldw=(1 << 22) + 16), dict(ls=1), dict(ldx=-100)])
def test_linear_refuses_past_its_limits(lib, bad):
    from spider_moe_amd import _native as nat

    def go(ldx=100, n=40, k=100, ldw=64, ls=4, no=30):
        return lib.smoe_linear_mxfp4(FAKE, nat.BF16, ldx, n, k, FAKE, ldw, FAKE, ls, None, no, 0, FAKE, nat.BF16, FAKE,
                                     1 << 40, None)

    assert go(n=0) == 0  # the call itself is sound
    assert go(**bad) == 1
    assert go(**{**bad, "n": 1}) == 1  # a few rows as well


def test_linear_workspace_at_the_limits(lib):
    f = lib.smoe_linear_mxfp4_workspace_bytes
    k, no = 1 << 23, 1 << 22
    assert f(40, k, 64) >= 40 * (k // 2 + k // 32)
    assert f(40, k + 1, 64) == 0 and f(40, 64, no + 1) == 0 and f(40, 64, no) > 0


def test_expert_limits(lib):
    from spider_moe_amd import _native as nat

    def need(n=30, k=2, e=4, h=64, u=96):
        d = nat.SmoeExpertsMxfp4()
        d.act, d.E, d.H, d.U = 0, e, h, u
        d.w_up = d.w_down = d.s_up = d.s_down = FAKE
        return lib.smoe_expert_delta_mxfp4_workspace_bytes(ctypes.byref(d), n, k)

    top = 1 << 22
    assert need(h=top, u=1024) > 0 and need(h=1024, u=top) > 0    # U * H = 2^32
    assert need(h=top, u=1056) == 0 and need(h=1056, u=top) == 0
    assert need(h=top + 32, u=32) == 0 and need(h=32, u=top + 32) == 0
    assert need(n=1024, k=1, h=top, u=32) > 0                      # N * H = 2^32
    assert need(n=1025, k=1, h=top, u=32) == 0
