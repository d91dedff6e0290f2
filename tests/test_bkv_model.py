"""The block-scaled cache's restatement (tests/bkv_model.py) against the formats'
definitions, and the C entry points' refusals that need no device."""
import ctypes as C

import numpy as np
import pytest

from tests import bkv_model as bm
from vokra_amd import hip


def test_e4m3_matches_the_table_of_its_values():
    """Nearest of all 253 finite values, ties to the even mantissa."""
    vals = []
    for code in range(0, 0x7f):
        e, m = code >> 3, code & 7
        vals.append((m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7))
    vals = np.array(vals)  # code order = value order
    g = np.random.default_rng(0)
    mids = (vals[:-1] + vals[1:]) / 2
    y = np.concatenate([vals, mids, np.nextafter(mids, 0), np.nextafter(mids, 1e9), np.exp(g.uniform(-8, 6.1, 4000))])
    y = y[y <= 448]
    i = np.clip(np.searchsorted(vals, y), 1, len(vals) - 1)
    lo, hi = vals[i - 1], vals[i]
    even = np.where((i - 1) % 2 == 0, lo, hi)
    want = np.where(y - lo < hi - y, lo, np.where(y - lo > hi - y, hi, even))
    # a value of the table is its own nearest
    want = np.where(y == hi, hi, np.where(y == lo, lo, want))
    assert np.array_equal(bm.e4m3(y), want)
    assert np.array_equal(bm.e4m3(-y), -want)


@pytest.mark.parametrize("codec", [0, 1])
def test_a_value_is_off_by_half_a_step_at_most(codec):
    """int8: half a step of a / 127 (and the f32 roundings); e4m3: 2^-4 of the
    value, half the smallest step near zero."""
    x = np.random.default_rng(1).standard_normal((16, 3, 64)).astype(np.float32) * 7
    y = bm.held_block(x, codec)
    a = np.abs(x).max((0, 2), keepdims=True).astype(np.float64)
    err = np.abs(y.astype(np.float64) - x)
    if codec == 0:
        assert np.all(err <= a / 127 * 0.5 * (1 + 1e-4))
    else:
        assert np.all(err <= np.maximum(np.abs(x) * 2.0 ** -4, a / 448 * 2.0 ** -10) * (1 + 1e-4))


def test_blocks_of_zeros_tiny_and_not_finite_values():
    x = np.zeros((16, 4, 64), np.float32)
    x[3, 1, 5] = 2.0 ** -101
    x[4, 2, 6] = np.inf
    x[5, 3, 7] = np.nan
    y = bm.held_block(x, 0)
    assert np.all(y[:, :2] == 0) and np.all(np.isnan(y[:, 2:]))


NULL = C.c_void_p()
CALLS = {
    "create": (NULL, 1, 1, 64, 1, 16, 16, 1, 1, 0, C.byref(C.c_void_p())),
    "reset": (NULL, NULL),
    "step": (NULL, NULL, 0, None, None, None),
    "step_dev": (NULL, NULL, 0, 0, 0, 0, NULL, NULL, NULL),
    "status": (NULL, NULL, None),
    "write": (NULL, NULL, 0, None, None),
    "write_dev": (NULL, NULL, 0, NULL, NULL),
    "attn": (NULL, NULL, 0, 1, None, 1.0, None),
    "attn_dev": (NULL, NULL, 0, 1, NULL, 1.0, NULL),
    "read": (NULL, NULL, 0, 0, None, None, None, None),
    "read_dev": (NULL, NULL, 0, 0, NULL, NULL, NULL, NULL),
    "fork": (NULL, NULL, 0, None, None),
    "fork_dev": (NULL, NULL, 0, NULL, NULL),
    "free": (NULL, NULL, 0, None),
    "free_dev": (NULL, NULL, 0, NULL),
    "copy": (NULL, NULL, NULL, 0, None, None),
    "copy_dev": (NULL, NULL, NULL, 0, NULL, NULL),
    "compact": (NULL, NULL),
    "length": (NULL, NULL, 0, None),
    "pages": (NULL, NULL, None, None),
    "page_of": (NULL, NULL, 0, 0, None),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_a_missing_context_or_cache_is_refused(name):
    assert getattr(hip.lib(), f"vokra_hip_bkv_{name}")(*CALLS[name]) == 5
    hip.lib().vokra_hip_bkv_destroy(None)
