"""A call of the packed attention or the beam selection that finds no memory leaves nothing behind."""
import ctypes as C

import numpy as np
import pytest

from vokra_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def test_calls_after_an_allocation_that_failed(ctx):
    """Sizes that no card holds, refused by the allocation (none of it is touched)."""
    L = hip.lib()
    wide = ctx.packed_attn(1, 1 << 20, 64, 1024, 1, 64)
    many = ctx.beam_select(256, 32, 1 << 24, 1)
    small, pick = ctx.packed_attn(2, 8, 8, 2, 1, 64), ctx.beam_select(1, 2, 8, 2)
    far = C.cast(1 << 46, C.POINTER(C.c_float))  # never read
    off = np.array([0, 1 << 20], np.int32)
    koff = np.array([0, 1], np.int32)
    s, t = np.zeros(8192, np.float32), np.zeros((3, 8192), np.int32)
    sp, ip = hip._ptr(s, C.c_float), [hip._ptr(a, C.c_int32) for a in t]
    out = np.zeros(8192, np.float32)

    def works():
        q = np.ones((3, 128), np.float32)
        v = np.arange(192, dtype=np.float32).reshape(3, 64)
        got = small.attn(q, q[:, :64], v, [3], causal=True)
        assert np.allclose(got[0], np.tile(v[0], 2)) and np.allclose(got[2], np.tile(v[1], 2))
        assert pick.select(np.eye(2, 8, dtype=np.float32)[None], np.zeros((1, 2)), 2)[2].tolist() == [[0, 1]]

    for name, call in (
            ("plan", lambda: L.vokra_hip_packed_attn_create(ctx._h, 1, 1 << 20, 1 << 20, 1024, 1024, 128,
                                                            C.byref(C.c_void_p()))),
            ("attention", lambda: L.vokra_hip_packed_attn(ctx._h, wide._h, 1, hip._ptr(off, C.c_int32),
                                                          hip._ptr(koff, C.c_int32), far, far, far, 1.0, 0, 0, far)),
            ("selection", lambda: L.vokra_hip_beam_select(ctx._h, many._h, 256, 32, 1 << 24, 1, far, sp, None, -1,
                                                          hip._ptr(out, C.c_float), ip[0], ip[1], ip[2]))):
        print("[case] failed allocation", name, flush=True)
        works()
        assert call() not in (0, 5)
        works()
