"""Logits rules at the ends of what a call takes."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_logits_rules import F, _up, rules, same
from vokra_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


class _Long:
    """A device list of 2^31 - 1 entries of which the last ones are `a`."""

    N = 2 ** 31 - 1

    def __init__(self, ctx, a):
        self.b = hip.DeviceBuffer(ctx, 4 * self.N)
        self.ptr = self.b.ptr
        end = C.c_void_p(self.ptr.value + 4 * (self.N - a.size))
        assert hip.lib().vokra_hip_memcpy_htod(ctx._h, end, a.ctypes.data_as(C.c_void_p), a.nbytes) == 0


def test_rows_at_the_end_of_the_longest_lists(ctx):
    """Rows whose tokens and biases are the last of 2^31 - 1: places beyond the list
    are not read."""
    print("[case] rules longest lists", flush=True)
    g = np.random.default_rng(8)
    rows, vocab, n = 2, 9001, 5000
    x = g.standard_normal((rows, vocab)).astype(F)
    hist, ids = (g.integers(-3, vocab + 3, rows * n).astype(np.int32) for _ in (0, 1))
    val = g.standard_normal(rows * n).astype(F)
    cut = np.array([0, n, 2 * n])
    off = _up(ctx, (_Long.N - 2 * n + cut).astype(np.int32))
    ru = hip.LogitsRules(n_hist=_Long.N, hist=_Long(ctx, hist), hist_offsets=off, repetition=_up(ctx, np.full(rows, 1.5, F)),
                         n_bias=_Long.N, bias_ids=_Long(ctx, ids), bias=_Long(ctx, val), bias_offsets=off)
    out, nxt = _up(ctx, x), _up(ctx, np.zeros(rows, np.int32))
    ctx.logits_rules_dev(rows, vocab, _up(ctx, x), ru, out, nxt)
    ctx.synchronize()
    got = out.download(F, x.size).reshape(x.shape), nxt.download(np.int32, rows)
    same(got, rules(x, history=list(hist.reshape(rows, n)), repetition=[1.5] * rows,
                    biases=[list(zip(i, v)) for i, v in zip(ids.reshape(rows, n), val.reshape(rows, n))]))


def test_mask_strides_beyond_every_mask_are_refused(ctx):
    """A stride whose bytes leave 64 bits, on the device and on the host."""
    print("[case] rules mask stride", flush=True)
    x, nxt, mask = np.zeros((3, 40), F), np.zeros(3, np.int32), np.zeros(2, np.uint32)
    d, d_next, d_mask = _up(ctx, x), _up(ctx, nxt), _up(ctx, mask)
    for stride in (1, (1 << 40) + 1, 1 << 61, 2 ** 63):
        with pytest.raises(hip.InvalidArgument):
            ctx.logits_rules_dev(3, 40, d, hip.LogitsRules(mask=d_mask, mask_stride=stride), d, d_next)
        c = hip._LogitsRules()
        c.mask, c.mask_stride = mask.ctypes.data, stride
        assert hip.lib().vokra_hip_logits_rules(ctx._h, 3, 40, hip._ptr(x, C.c_float), C.byref(c),
                                                hip._ptr(x, C.c_float), hip._ptr(nxt, C.c_int32)) == 5
