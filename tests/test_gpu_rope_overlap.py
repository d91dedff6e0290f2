"""Which overlaps of buffers and sizes a rotary plan refuses, and rows that lie between each
other without overlapping."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_rope_plan import _At, check, thetas
from vokra_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def test_outputs_that_overlap_the_other_side_are_refused(ctx):
    print("[case] rope overlap", flush=True)
    plan = ctx.rope_plan(64, 64)
    buf = lambda n=8192: hip.DeviceBuffer.from_array(ctx, np.zeros(n, np.float32))  # noqa: E731
    a, b, c, pos = buf(), buf(), buf(), hip.DeviceBuffer.from_array(ctx, np.zeros(4, np.int32))
    n, row = 4, dict(q_stride=256, k_stride=256)
    for call in (lambda: plan.apply_dev(n, pos, 1, a, b, 1, b, c),  # q's output is k
                 lambda: plan.apply_dev(n, pos, 1, a, c, 1, b, a),  # k's output is q
                 lambda: plan.apply_dev(n, pos, 1, a, c, 1, b, c),  # one output for both
                 lambda: plan.apply_dev(n, pos, 1, a, c, 1, b, _At(c, 4 * 64 - 1)),
                 lambda: plan.apply_dev(n, pos, 1, a, _At(b, 4 * 64 - 1), 1, b, c),
                 lambda: plan.apply_dev(n, pos, 1, a, a, 1, a, a),  # both in place in one buffer
                 lambda: plan.apply_dev(n, pos, 2, a, a, 1, _At(a, 127), _At(a, 127), **row),
                 lambda: plan.apply_dev(n, pos, 2, a, a, 1, _At(a, 256 - 63), _At(a, 256 - 63), **row),
                 lambda: plan.apply_dev(n, pos, 2, a, _At(a, 127), q_stride=256, q_out_stride=256),
                 lambda: plan.apply_dev(n, a, 1, b, a), lambda: plan.apply_dev(n, a, 1, b, c, 1, a, a)):
        with pytest.raises(hip.InvalidArgument):
            call()


def test_rows_between_rows(ctx):
    """One buffer of rows [q | k | q's output | k's output]: nothing overlaps."""
    print("[case] rope rows between rows", flush=True)
    g = np.random.default_rng(4)
    n, hq, hk, hd = 33, 3, 2, 64
    wq, wk = hq * hd, hk * hd
    width = 2 * (wq + wk)
    rows = g.standard_normal((n, width)).astype(np.float32)
    pos = g.integers(0, 5000, n).astype(np.int32)
    b = hip.DeviceBuffer.from_array(ctx, rows)
    at = [_At(b, o) for o in (0, wq, wq + wk, 2 * wq + wk)]
    ctx.rope_plan(hd, hd).apply_dev(n, hip.DeviceBuffer.from_array(ctx, pos), hq, at[0], at[2], hk, at[1], at[3],
                                    q_stride=width, q_out_stride=width, k_stride=width, k_out_stride=width)
    ctx.synchronize()
    got = b.download(np.float32, rows.size).reshape(rows.shape)
    assert np.array_equal(got[:, :wq + wk], rows[:, :wq + wk])
    x = np.ascontiguousarray(rows[:, :wq + wk]).reshape(n, hq + hk, hd)
    check(np.ascontiguousarray(got[:, wq + wk:]), x, pos, thetas(hd, 10000.0), hip.RopeLayout.HALF)


def test_sizes_beyond_a_call_are_refused_before_any_copy(ctx):
    """Sizes whose product leaves 64 bits, too: nothing of the (short) arrays is read."""
    print("[case] rope sizes", flush=True)
    x, pos = np.zeros(64, np.float32), np.zeros(1, np.int32)
    f, i = hip._ptr(x, C.c_float), hip._ptr(pos, C.c_int32)
    for hd in (64, 65536):
        plan = ctx.rope_plan(hd, 64)
        for rows, hq, hk in ((2 ** 31 - 1, 65535, 65535), (2 ** 31, 1, 0), (1, 70000, 0), (1 << 27, 1, 1 if hd > 64 else 64)):
            assert hip.lib().vokra_hip_rope_apply(ctx._h, plan._h, rows, i, hq, f, f, hk, f, f) == 5
