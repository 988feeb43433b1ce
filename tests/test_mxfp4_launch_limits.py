"""Microscaled 4-bit products past a launch's limits are refused before anything
is launched (CPU: a launch would fail here with another status), and the limits
are those that include/smoe.h states."""
import ctypes

import pytest

FAKE = 0x1000  # never dereferenced: every call below is refused
EINVAL = 1


@pytest.fixture(scope="module")
def lib():
    from spider_moe_amd import _native
    return _native.lib()


def linear(lib, n, k, n_out):
    from spider_moe_amd import _native as nat
    ldw, ls = 16 * -(-k // 32), 4 * -(-k // 128)
    return lib.smoe_linear_mxfp4(FAKE, nat.BF16, k, n, k, FAKE, ldw, FAKE, ls, None, n_out, 0, FAKE, nat.BF16, FAKE,
                                 1 << 62, None)


def experts(lib, n, k, e, h, u, act=0):
    from spider_moe_amd import _native as nat
    d = nat.SmoeExpertsMxfp4()
    d.act, d.E, d.H, d.U = act, e, h, u
    d.w_up = d.w_down = d.s_up = d.s_down = FAKE
    need = lib.smoe_expert_delta_mxfp4_workspace_bytes(ctypes.byref(d), n, k)
    return need, lib.smoe_expert_delta_mxfp4(ctypes.byref(d), FAKE, nat.BF16, FAKE, FAKE, n, k, FAKE, nat.BF16, FAKE,
                                             1 << 62, None)


def test_linear_tiles(lib):
    assert linear(lib, 1 << 24, 32, 1 << 22) == EINVAL  # 2^31 tiles
    assert b"tiles" in lib.smoe_last_error()
    assert linear(lib, 1 << 28, 1, 1) == EINVAL         # 2^28 pieces of rows
    assert linear(lib, 1 << 14, (1 << 21) + 1, 64) == EINVAL


def test_linear_weight_pieces(lib):
    f = lib.smoe_linear_mxfp4_workspace_bytes
    assert f(40, 1 << 17, 1 << 22) == 0 and f(40, (1 << 17) - 128, 1 << 22) > 0  # 2^32 pieces; 2^22 fewer
    assert linear(lib, 40, 1 << 17, 1 << 22) == EINVAL and b"2^32 - 512" in lib.smoe_last_error()


@pytest.mark.parametrize("n,k,e,h,u", [
    (1024, 16, 256, 32, 1 << 22),   # up to 64 rows an expert, 32-row tiles: 2^25 workgroups
    (1024, 1, 256, 1 << 20, 32),    # a streamed down product of 256 * 2^16 strips, 16 channels each
])
def test_expert_tiles(lib, n, k, e, h, u):
    need, rc = experts(lib, n, k, e, h, u)
    assert need > 0 and rc == EINVAL and b"tiles" in lib.smoe_last_error()


def test_expert_weight_pieces(lib):
    size = dict(e=256, h=160, u=(1 << 22) - 32)  # two words a row of 160: 2^32 words of gates and ups
    assert experts(lib, 4096, 32, **size, act=1) == (0, EINVAL)
    assert b"2^32 - 512" in lib.smoe_last_error()
