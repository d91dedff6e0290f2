"""A call that finds no memory leaves nothing behind: the next one runs."""
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
    x, pos = np.ones(64, np.float32), np.zeros(1, np.int32)
    f, i = hip._ptr(x, C.c_float), hip._ptr(pos, C.c_int32)
    kv, plan = ctx.block_kv_cache(1, 2, 64, 2, 100, 16, 10, 64), ctx.rope_plan(65536, 64)
    L = hip.lib()
    n = 2 ** 31 - 1

    def works():
        kv.step([0], [kv.length(0)], [1])
        kv.write(0, x.repeat(2), x.repeat(2))
        assert np.all(kv.read(0, [0], [0])[0] == 1)
        assert np.array_equal(ctx.rope_plan(64, 64).apply([0], x)[0], x)
        assert list(ctx.logits_rules(np.eye(3, dtype=np.float32))[1]) == [0, 1, 2]
        assert np.array_equal(ctx.rms_norm_f32(x, 1, 64, x, 0.0).reshape(-1), x)

    for name, call in (("read", lambda: L.vokra_hip_bkv_read(ctx._h, kv._h, 0, n, i, i, f, f)),
                       ("create", lambda: L.vokra_hip_bkv_create(ctx._h, 4096, 1024, 128, 65535, 1 << 24, 64, 1 << 26, 1,
                                                                 0, C.byref(C.c_void_p()))),
                       ("rules", lambda: L.vokra_hip_logits_rules(
                           ctx._h, 65535, 1 << 24, f, C.byref(hip._LogitsRules()), f, i)),
                       ("device_alloc", lambda: L.vokra_hip_device_alloc(ctx._h, 1 << 43, C.byref(C.c_void_p())))):
        print("[case] failed allocation", name, flush=True)
        works()
        assert call() not in (0, 5)
        works()
