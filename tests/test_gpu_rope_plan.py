"""GPU parity of rotary plans with the rotation in extended precision."""
import ctypes as C

import numpy as np
import pytest

from vokra_amd import hip

LD = np.longdouble
TWO_PI = LD("6.283185307179586476925286766559")
HALF, PAIRS = hip.RopeLayout.HALF, hip.RopeLayout.INTERLEAVED
SC = hip.RopeScaling


def thetas(rot, base, scaling=SC.NONE, factor=1.0, orig=0, fast=32.0, slow=1.0, low=1.0, high=4.0, divisors=None):
    j = np.arange(rot // 2, dtype=LD)
    if scaling == SC.NTK:
        return (LD(base) * LD(factor) ** (LD(rot) / LD(rot - 2))) ** (-2 * j / rot)
    th = LD(base) ** (-2 * j / rot)
    if scaling == SC.LINEAR:
        return th / LD(factor)
    if scaling == SC.DIVISORS:
        return th / np.asarray(divisors, LD)
    if scaling == SC.YARN:
        def d(t):
            return rot * np.log(LD(orig) / (LD(t) * TWO_PI)) / (2 * np.log(LD(base)))
        lo, hi = max(np.floor(d(fast)), LD(0)), min(np.ceil(d(slow)), LD(rot - 1))
        r = np.clip((j - lo) / max(hi - lo, LD("0.001")), 0, 1)
        return th / LD(factor) * r + th * (1 - r)
    if scaling == SC.BANDS:
        m = np.clip((LD(orig) * th / TWO_PI - LD(low)) / (LD(high) - LD(low)), 0, 1)
        return th / LD(factor) * (1 - m) + th * m
    return th


def rotate(x, pos, th, layout, mag):
    """(rotated, bound): x [n, heads, hd]. The bound: the rest of the angle is
    held to 2^-33 of a turn and rounded twice (below pi / 4), the polynomials to
    a few roundings, the magnitude and the two products to one each: 8 units of
    2^-24 of (|a| + |b|) magnitude."""
    rot = 2 * th.size
    turns = (np.asarray(pos, LD)[:, None] * th) / TWO_PI
    ang = (turns - np.floor(turns)) * TWO_PI
    c, s = (f(ang)[:, None] * LD(mag) for f in (np.cos, np.sin))
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == HALF else (slice(0, rot, 2), slice(1, rot, 2))
    y, tol = x.astype(LD), np.zeros(x.shape)
    a, b = x[..., i].astype(LD), x[..., j].astype(LD)
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    tol[..., i] = tol[..., j] = (np.abs(a) + np.abs(b)) * mag * 8 * 2.0 ** -24
    return y, tol


def check(got, x, pos, th, layout, mag=1.0):
    want, tol = rotate(x, pos, th, layout, mag)
    err = np.abs(got.reshape(x.shape).astype(LD) - want)
    assert np.all(err <= tol), float((err - tol).max())


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("hd,rot,hq,hk,n", [(128, 128, 16, 2, 33), (64, 32, 3, 3, 5), (80, 20, 2, 1, 7), (96, 72, 5, 0, 4),
                                            (256, 2, 1, 1, 3), (6, 4, 2, 2, 9), (128, 64, 0, 4, 1), (10, 10, 1, 1, 65)])
def test_layouts_and_parts_of_the_head(ctx, layout, hd, rot, hq, hk, n):
    print("[case] rope", layout, hd, rot, hq, hk, n, flush=True)
    g = np.random.default_rng(hd + n)
    pos = g.integers(0, 5000, n).astype(np.int32)
    plan = ctx.rope_plan(hd, rot, layout, 10000.0)
    q, k = (g.standard_normal((n, h * hd)).astype(np.float32) if h else None for h in (hq, hk))
    for got, x, h in zip(plan.apply(pos, q, k), (q, k), (hq, hk)):
        if h:
            check(got, x.reshape(n, h, hd), pos, thetas(rot, 10000.0), layout)


@pytest.mark.gpu
def test_positions_near_and_far(ctx):
    print("[case] rope far", flush=True)
    pos = np.array([0, 1, -1, 131071, 1000003, 2 ** 24 + 1, -7654321, 2 ** 31 - 1, -2 ** 31], np.int32)
    x = np.random.default_rng(0).standard_normal((pos.size, 2 * 128)).astype(np.float32)
    for base in (1.5, 10000.0, 500000.0):
        got, _ = ctx.rope_plan(128, 128, HALF, base).apply(pos, x)
        check(got, x.reshape(-1, 2, 128), pos, thetas(128, base), HALF)
    assert np.array_equal(ctx.rope_plan(128, 64, HALF).apply(pos[:1], x[:1])[0], x[:1])  # position 0 turns nothing


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [
    dict(scaling=SC.LINEAR, factor=4.0), dict(scaling=SC.NTK, factor=8.0),
    dict(scaling=SC.YARN, factor=8.0, orig=4096), dict(scaling=SC.YARN, factor=2.5, orig=100, fast=8.0, slow=2.0),
    dict(scaling=SC.BANDS, factor=8.0, orig=8192), dict(scaling=SC.BANDS, factor=3.0, orig=50, low=0.5, high=7.0),
    dict(scaling=SC.DIVISORS, divisors=np.linspace(1, 30, 48))])
def test_scalings(ctx, kw):
    print("[case] rope scaling", kw["scaling"], flush=True)
    g = np.random.default_rng(1)
    pos = g.integers(0, 200000, 50).astype(np.int32)
    x = g.standard_normal((50, 3 * 128)).astype(np.float32)
    names = {"orig": "orig_ctx", "fast": "beta_fast", "slow": "beta_slow", "low": "low_turns", "high": "high_turns"}
    plan = ctx.rope_plan(128, 96, PAIRS, 500000.0, **{names.get(k, k): v for k, v in kw.items()})
    mag = 0.1 * np.log(kw["factor"]) + 1 if kw["scaling"] == SC.YARN else 1.0
    check(plan.apply(pos, x)[0], x.reshape(50, 3, 128), pos, thetas(96, 500000.0, **kw), PAIRS, mag)
    plan = ctx.rope_plan(128, 96, PAIRS, 500000.0, magnitude=0.7, **{names.get(k, k): v for k, v in kw.items()})
    check(plan.apply(pos, x)[0], x.reshape(50, 3, 128), pos, thetas(96, 500000.0, **kw), PAIRS, 0.7)


class _At:
    def __init__(self, buf, floats):
        self.ptr = C.c_void_p(buf.ptr.value + 4 * floats)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("hd,rot,n,shift", [(64, 48, 9, 0), (64, 48, 9, 1), (128, 128, 700, 0), (80, 20, 3, 4), (64, 64, 5, 2)])
def test_strided_rows_in_place_and_out(ctx, layout, hd, rot, n, shift):
    """q and k inside one projection's rows, at any float offset: in place nothing
    else changes, out of place the inputs stay and rows beyond are not written."""
    print("[case] rope strides", layout, hd, rot, n, shift, flush=True)
    hq, hk = 3, 2
    g = np.random.default_rng(3)
    width = (hq + 2 * hk) * hd + 4 + shift
    rows = g.standard_normal((n, width)).astype(np.float32)
    pos = g.integers(0, 100000, n).astype(np.int32)
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    qkv, d_pos = up(np.r_[rows.reshape(-1), np.zeros(8, np.float32)]), up(pos)
    plan, th = ctx.rope_plan(hd, rot, layout), thetas(rot, 10000.0)
    q, k = _At(qkv, shift), _At(qkv, shift + hq * hd)
    wq, wk = hq * hd + 3, hk * hd + 4
    qo, ko = up(np.full((n + 1) * wq, 9.0, np.float32)), up(np.full((n + 1) * wk, 9.0, np.float32))
    plan.apply_dev(n, d_pos, hq, q, qo, hk, k, ko, q_stride=width, k_stride=width, q_out_stride=wq, k_out_stride=wk)
    ctx.synchronize()
    flat = np.r_[rows.reshape(-1), np.zeros(8, np.float32)]
    assert np.array_equal(qkv.download(np.float32, flat.size), flat)
    cut = [np.lib.stride_tricks.as_strided(flat[o:], (n, h, hd), (4 * width, 4 * hd, 4)) for o, h in
           ((shift, hq), (shift + hq * hd, hk))]
    for buf, w, h, x in ((qo, wq, hq, cut[0]), (ko, wk, hk, cut[1])):
        got = buf.download(np.float32, (n + 1) * w).reshape(n + 1, w)
        check(np.ascontiguousarray(got[:n, :h * hd]), np.ascontiguousarray(x), pos, th, layout)
        assert np.all(got[:, h * hd:] == 9.0) and np.all(got[n] == 9.0)
    plan.apply_dev(n, d_pos, hq, q, q, hk, k, k, q_stride=width, k_stride=width)
    ctx.synchronize()
    after = qkv.download(np.float32, flat.size)
    want = flat.copy()
    for o, buf, w, h in ((shift, qo, wq, hq), (shift + hq * hd, ko, wk, hk)):
        view = np.lib.stride_tricks.as_strided(want[o:], (n, h * hd), (4 * width, 4))
        view[:] = buf.download(np.float32, (n + 1) * w).reshape(n + 1, w)[:n, :h * hd]
    assert np.array_equal(after, want)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [HALF, PAIRS])
def test_more_rows_than_the_caches_hold(ctx, layout):
    """One call over 34 million values and the same rows in three: equal bits."""
    print("[case] rope large", layout, flush=True)
    n, h, hd = 4101, 64, 128
    g = np.random.default_rng(9)
    x = g.random((n, h * hd), np.float32) - np.float32(0.5)
    pos = g.integers(0, 200000, n).astype(np.int32)
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    d, dp, whole, parts = up(x), up(pos), up(np.zeros_like(x)), up(np.zeros_like(x))
    plan = ctx.rope_plan(hd, 64, layout)
    plan.apply_dev(n, dp, h, d, whole)
    for a, b in ((0, 1400), (1400, 2800), (2800, n)):
        plan.apply_dev(b - a, _At(dp, a), h, _At(d, a * h * hd), _At(parts, a * h * hd))
    ctx.synchronize()
    got = whole.download(np.float32, x.size)
    assert np.array_equal(got, parts.download(np.float32, x.size))
    some = [0, 2047, n - 1]
    check(got.reshape(n, -1)[some], x[some].reshape(3, h, hd), pos[some], thetas(64, 10000.0), layout)


@pytest.mark.gpu
def test_a_captured_turn_takes_the_positions_of_its_replay(ctx):
    print("[case] rope graph", flush=True)
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    x = np.random.default_rng(0).standard_normal((4, 2 * 64)).astype(np.float32)
    d, o, pos = up(x), up(np.zeros_like(x)), up(np.zeros(4, np.int32))
    plan = ctx.rope_plan(64, 64)
    graph = ctx.capture(lambda: plan.apply_dev(4, pos, 2, d, o))
    for i in range(4):
        p = np.arange(4, dtype=np.int32) * 1000 * i + i
        pos.upload(p)
        graph.launch()
        ctx.synchronize()
        check(o.download(np.float32, x.size), x.reshape(4, 2, 64), p, thetas(64, 10000.0), HALF)
        assert np.array_equal(o.download(np.float32, x.size), plan.apply(p, x)[0].reshape(-1))


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] rope refusals", flush=True)
    inf, nan = float("inf"), float("nan")
    for args, kw in (((64, 0), {}), ((64, 3), {}), ((64, 66), {}), ((0, 0), {}), ((64, 64, 7), {}),
                     ((64, 64, 0, 1.0), {}), ((64, 64, 0, inf), {}), ((64, 64, 0, nan), {}), ((64, 64, 0, 10.0, 9), {}),
                     ((64, 64, 0, 10.0, SC.LINEAR, 0.5), {}), ((64, 64, 0, 10.0, SC.LINEAR, nan), {}),
                     ((64, 2, 0, 10.0, SC.NTK, 2.0), {}), ((64, 64, 0, 10.0, SC.YARN, 2.0, 0), {}),
                     ((64, 64, 0, 10.0, SC.YARN, 2.0, 9), dict(beta_fast=-1.0)),
                     ((64, 64, 0, 10.0, SC.BANDS, 2.0, 9), dict(low_turns=4.0, high_turns=4.0)),
                     ((64, 64), dict(magnitude=-1.0)), ((64, 64, 0, 10.0, SC.DIVISORS), {}),
                     ((64, 64, 0, 10.0, SC.DIVISORS), dict(divisors=np.zeros(32))),
                     ((64, 64, 0, 10.0, SC.DIVISORS), dict(divisors=np.ones(31)))):
        with pytest.raises(hip.InvalidArgument):
            ctx.rope_plan(*args, **kw)
    plan = ctx.rope_plan(64, 64)
    b = hip.DeviceBuffer.from_array(ctx, np.zeros(4096, np.float32))
    o = hip.DeviceBuffer.from_array(ctx, np.zeros(4096, np.float32))
    null = type("P", (), {"ptr": C.c_void_p()})()
    for call in (lambda: plan.apply_dev(2, null, 1, b, o), lambda: plan.apply_dev(2, b, 1, null, o),
                 lambda: plan.apply_dev(2, b, 1, b, null), lambda: plan.apply_dev(2, b, 1, b, o, q_stride=63),
                 lambda: plan.apply_dev(2, b, 1, b, b, q_stride=64, q_out_stride=65),
                 lambda: plan.apply_dev(2, b, 1, b, _At(b, 4)), lambda: plan.apply_dev(2, b, 0, None, None, 1, b, null),
                 lambda: plan.apply_dev(2, b, 70000, b, o), lambda: plan.apply_dev(2 ** 31, b, 1, b, o),
                 lambda: plan.apply([0], np.zeros(63, np.float32))):
        with pytest.raises(hip.InvalidArgument):
            call()
    plan.apply_dev(0, null, 1, b, o)
    plan.apply_dev(2, null, 0, None, None)


def test_missing_arguments_are_refused_without_a_device():
    L, null = hip.lib(), C.c_void_p()
    assert L.vokra_hip_rope_create(null, None, C.byref(C.c_void_p())) == 5
    assert L.vokra_hip_rope_apply_dev(null, null, 1, null, 1, null, 1, null, 1, 0, null, 0, null, 0) == 5
    assert L.vokra_hip_rope_apply(null, null, 1, None, 1, None, None, 0, None, None) == 5
    L.vokra_hip_rope_destroy(None)
