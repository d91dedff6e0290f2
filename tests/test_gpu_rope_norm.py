"""GPU parity of head norms with their rotation against the formula in extended precision."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_rope_plan import HALF, LD, PAIRS, SC, rotate, thetas
from vokra_amd import hip


def normed(x, gamma, eps):
    """x [n, heads, hd] by the root of its mean square and gamma, and a head's rounding
    units of 2^-24: a lane adds up to max(8, hd / 64) squares (a product each), lanes join
    in at most six steps, the mean takes two roundings and eps one; the root halves what
    came before and rounds once, as do the division and the two products."""
    x = x.astype(LD)
    hd = x.shape[-1]
    y = x / np.sqrt((x * x).sum(-1, keepdims=True) / hd + LD(np.float32(eps)))
    units = (max(8, -(-hd // 64)) + 1 + 6 + 3) / 2 + 4
    return (y if gamma is None else y * gamma.astype(LD)), units


def check(got, x, gamma, eps, pos, th, layout, mag=1.0):
    y, units = normed(x, gamma, eps)
    want, tol = rotate(y, pos, th, layout, mag)
    # rotate's 8 units on the pair, and the norm's on each of its values; beyond the rotation the norm's alone
    tol = tol * (8 + units) / 8
    rot = 2 * th.size
    tol[..., rot:] = np.abs(y[..., rot:]) * units * 2.0 ** -24
    err = np.abs(got.reshape(x.shape).astype(LD) - want)
    assert np.all(err <= tol), float((err - tol).max())


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [HALF, PAIRS])
@pytest.mark.parametrize("hd,rot,hq,hk,n", [
    (128, 128, 16, 2, 33), (64, 32, 3, 3, 5), (80, 24, 2, 1, 7), (96, 96, 5, 0, 4), (256, 8, 1, 1, 3), (8, 8, 2, 2, 9),
    (16, 8, 1, 2, 70), (24, 16, 3, 1, 2), (512, 512, 2, 1, 3), (128, 64, 0, 4, 1),  # the vector kernel's groups of lanes
    (80, 20, 2, 1, 7), (6, 4, 2, 2, 9), (10, 10, 1, 1, 65), (1000, 504, 1, 2, 3), (2, 2, 1, 1, 5)])  # any size
def test_layouts_and_sizes(ctx, layout, hd, rot, hq, hk, n):
    print("[case] rope norm", layout, hd, rot, hq, hk, n, flush=True)
    g = np.random.default_rng(hd + n)
    pos = g.integers(0, 5000, n).astype(np.int32)
    plan = ctx.rope_plan(hd, rot, layout, 10000.0)
    q, k = ((g.standard_normal((n, h * hd)) * np.exp(g.normal(0, 3, (n, 1)))).astype(np.float32) if h else None
            for h in (hq, hk))
    for per_head in (False, True):
        gq, gk = (g.normal(1, 0.5, (h, hd) if per_head else hd).astype(np.float32) if h else None for h in (hq, hk))
        for eps in (1e-5, 0.0):
            got = plan.norm_apply(pos, eps, q, gq, k, gk)
            for y, x, gamma, h in zip(got, (q, k), (gq, gk), (hq, hk)):
                if h:
                    check(y, x.reshape(n, h, hd), gamma, eps, pos, thetas(rot, 10000.0), layout)
    for y, x, h in zip(plan.norm_apply(pos, 1e-6, q, None, k, None), (q, k), (hq, hk)):
        if h:
            check(y, x.reshape(n, h, hd), None, 1e-6, pos, thetas(rot, 10000.0), layout)


@pytest.mark.gpu
def test_many_rows_share_sines_and_scaled_plans(ctx):
    """More rows than one head a thread group takes; far positions; a magnitude."""
    print("[case] rope norm many", flush=True)
    g = np.random.default_rng(0)
    for n, hq, hk in ((1200, 12, 3), (2051, 32, 8)):
        pos = g.integers(-2 ** 31, 2 ** 31 - 1, n).astype(np.int32)
        q, k = (g.standard_normal((n, h * 128)).astype(np.float32) for h in (hq, hk))
        gq, gk = (g.normal(1, 0.3, 128).astype(np.float32) for _ in range(2))
        kw = dict(scaling=SC.YARN, factor=8.0, orig=4096)
        plan = ctx.rope_plan(128, 64, HALF, 500000.0, scaling=SC.YARN, factor=8.0, orig_ctx=4096)
        for y, x, gamma, h in zip(plan.norm_apply(pos, 1e-5, q, gq, k, gk), (q, k), (gq, gk), (hq, hk)):
            check(y, x.reshape(n, h, 128), gamma, 1e-5, pos, thetas(64, 500000.0, **kw), HALF, 0.1 * np.log(8.0) + 1)


def _up(ctx, a):
    return hip.DeviceBuffer.from_array(ctx, a)


class At:
    """A part of a device buffer, from float `at` on."""

    def __init__(self, buf, at):
        self.ptr, self.keep = C.c_void_p(buf.ptr.value + 4 * at), buf


@pytest.mark.gpu
@pytest.mark.parametrize("hd,shift,pad,in_place", [(128, 0, 0, True), (128, 0, 4, False), (64, 1, 0, True), (64, 0, 3, False),
                                                   (96, 2, 1, True), (128, 0, 8, True)])
def test_rows_of_a_projection(ctx, hd, shift, pad, in_place):
    """q and k as parts of one buffer's rows, aligned or not; what is no head stays."""
    print("[case] rope norm strides", hd, shift, pad, in_place, flush=True)
    g = np.random.default_rng(hd + pad)
    hq, hk, n = 6, 2, 21
    w = (hq + 2 * hk) * hd + pad
    x = g.standard_normal(n * w + shift).astype(np.float32)
    rows = x[shift:].reshape(n, w)
    pos = g.integers(0, 900, n).astype(np.int32)
    gq, gk = g.normal(1, 0.2, (hq, hd + 4)).astype(np.float32), g.normal(1, 0.2, hd).astype(np.float32)
    plan = ctx.rope_plan(hd, hd // 2, PAIRS)
    d_x, d_p, d_gq, d_gk = _up(ctx, x), _up(ctx, pos), _up(ctx, gq), _up(ctx, gk)
    q, k = At(d_x, shift), At(d_x, shift + hq * hd)
    kw = dict(q_gamma_stride=hd + 4, q_stride=w, k_stride=w)
    if in_place:
        plan.norm_apply_dev(n, d_p, 1e-5, hq, q, d_gq, q, hk, k, d_gk, k, **kw)
        out = d_x.download(np.float32, x.size)
        assert np.array_equal(out[:shift], x[:shift])
        out = out[shift:].reshape(n, w)
        assert np.array_equal(out[:, (hq + hk) * hd:], rows[:, (hq + hk) * hd:])
    else:
        d_o = _up(ctx, np.full((n, w), 7.0, np.float32))
        plan.norm_apply_dev(n, d_p, 1e-5, hq, q, d_gq, d_o, hk, k, d_gk, At(d_o, hq * hd), q_out_stride=w,
                            k_out_stride=w, **kw)
        assert np.array_equal(d_x.download(np.float32, x.size), x)
        out = d_o.download(np.float32, n * w).reshape(n, w)
        assert np.all(out[:, (hq + hk) * hd:] == 7.0)
    th = thetas(hd // 2, 10000.0)
    check(out[:, :hq * hd], rows[:, :hq * hd].reshape(n, hq, hd), gq[:, :hd], 1e-5, pos, th, PAIRS)
    check(out[:, hq * hd:(hq + hk) * hd], rows[:, hq * hd:(hq + hk) * hd].reshape(n, hk, hd), gk, 1e-5, pos, th, PAIRS)


@pytest.mark.gpu
def test_rows_of_zeros_and_values_that_are_not_finite(ctx):
    print("[case] rope norm edges", flush=True)
    for hd in (128, 10):  # both kernels
        plan = ctx.rope_plan(hd, hd)
        x = np.random.default_rng(0).standard_normal((5, 2, hd)).astype(np.float32)
        x[0] = 0.0
        x[1, 0, 3] = np.nan
        x[2, 1, 0] = np.inf
        x[3, 0] = 1e-30  # squares below f32: eps alone is left
        pos = np.arange(5, dtype=np.int32)
        y = plan.norm_apply(pos, 1e-5, x.reshape(5, -1))[0].reshape(x.shape)
        assert np.all(y[0] == 0.0)
        # a NaN is the whole head's, an infinity's pair is NaN, and the heads beside them do not change
        assert np.all(np.isnan(y[1, 0])) and np.isnan(y[2, 1, 0])
        for r, h in ((1, 1), (2, 0), (3, 0), (4, 0), (4, 1)):
            check(y[r:r + 1, h:h + 1], x[r:r + 1, h:h + 1], None, 1e-5, pos[r:r + 1], thetas(hd, 10000.0), HALF)


@pytest.mark.gpu
def test_in_a_graph(ctx):
    print("[case] rope norm graph", flush=True)
    g = np.random.default_rng(3)
    n, hq, hk, hd = 40, 8, 2, 128
    plan = ctx.rope_plan(hd, hd)
    gq = g.normal(1, 0.2, hd).astype(np.float32)
    d_q, d_k, d_p, d_g = (_up(ctx, a) for a in (np.zeros((n, hq * hd), np.float32), np.zeros((n, hk * hd), np.float32),
                                                np.zeros(n, np.int32), gq))
    d_qo, d_ko = hip.DeviceBuffer(ctx, n * hq * hd * 4), hip.DeviceBuffer(ctx, n * hk * hd * 4)
    ctx.synchronize()
    graph = ctx.capture(lambda: plan.norm_apply_dev(n, d_p, 1e-5, hq, d_q, d_g, d_qo, hk, d_k, None, d_ko))
    for i in range(3):
        q, k = (g.standard_normal((n, h * hd)).astype(np.float32) for h in (hq, hk))
        pos = g.integers(0, 10000, n).astype(np.int32)
        for d, a in ((d_q, q), (d_k, k), (d_p, pos)):
            d.upload(a)
        graph.launch()
        ctx.synchronize()
        got = d_qo.download(np.float32, q.size), d_ko.download(np.float32, k.size)
        for y, e in zip(got, plan.norm_apply(pos, 1e-5, q, gq, k, None)):
            assert np.array_equal(y, e.reshape(-1))


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] rope norm refusals", flush=True)
    plan = ctx.rope_plan(64, 64)
    b, p, gm = hip.DeviceBuffer(ctx, 16384), hip.DeviceBuffer(ctx, 256), hip.DeviceBuffer(ctx, 4096)
    o = hip.DeviceBuffer(ctx, 16384)

    def bad(*a, **kw):
        with pytest.raises(hip.InvalidArgument):
            plan.norm_apply_dev(*a, **kw)
    bad(4, p, float("nan"), 2, b, gm, o)
    bad(4, p, -1.0, 2, b, gm, o)
    bad(4, p, float("inf"), 2, b, gm, o)
    bad(4, p, 1e-5, 2, b, gm, o, q_gamma_stride=63)
    bad(4, p, 1e-5, 2, b, gm, o, q_gamma_stride=2 ** 41)
    bad(4, p, 1e-5, 2, None, gm, o)
    bad(4, p, 1e-5, 2, b, gm, At(b, 64))  # overlaps its input
    bad(4, p, 1e-5, 2, b, gm, gm)  # overlaps the weights
    bad(4, p, 1e-5, 2, b, At(o, 100), o)
    bad(4, p, 1e-5, 0, None, None, None, 2, b, At(o, 4 * 128 - 1), o)
    bad(4, p, 1e-5, 2, b, gm, o, q_stride=100)
    bad(4, At(o, 10), 1e-5, 2, b, gm, o)
    plan.norm_apply_dev(0, p, 1e-5, 2, b, gm, o)
    plan.norm_apply_dev(4, p, 1e-5, 2, b, At(o, 4 * 128), o)  # right behind
    with pytest.raises(hip.InvalidArgument):
        plan.norm_apply(np.arange(2), 1e-5, np.zeros((2, 128)), np.zeros(63))
    with pytest.raises(hip.InvalidArgument):
        plan.norm_apply(np.arange(2), 1e-5, np.zeros((2, 128)), np.zeros((3, 64)))
    ctx.synchronize()


def test_missing_arguments_are_refused_without_a_device():
    L = hip.lib()
    norm = hip._HeadNorm(eps=1e-5)
    for code in (L.vokra_hip_rope_norm_apply_dev(None, None, C.byref(norm), 1, None, 1, None, 1, None, 1, 0, None, 0,
                                                 None, 0),
                 L.vokra_hip_rope_norm_apply_dev(None, None, None, 1, None, 1, None, 1, None, 1, 0, None, 0, None, 0),
                 L.vokra_hip_rope_norm_apply(None, None, C.byref(norm), 1, None, 1, None, None, 0, None, None),
                 L.vokra_hip_rope_norm_apply(None, None, None, 1, None, 1, None, None, 0, None, None)):
        assert code == 5
        assert b"rope_" in L.vokra_hip_last_error()
