"""GPU parity of attention over packed sequences with the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from vokra_amd import hip

F = np.float32


def seen(n, m, causal, window):
    """[n, m]: which keys the rows see."""
    p = np.arange(n)[:, None] + (m - n)
    j = np.arange(m)[None]
    s = np.ones((n, m), bool)
    if causal:
        s = j <= p
        if window:
            s &= j > p - window
    return s


def attend(q, k, v, q_lens, k_lens, hq, hkv, scale, causal=False, window=0):
    """(outputs, bounds) [rows, hq, hd] in 64 bits. The bound: an operand's two fp16 parts hold it to
    2^-22 (half a step of each, 2^-11 of 2^-11), as much is left out with lo lo, so a product is off by
    3 * 2^-22 at most, and 3 hd of them are added in f32, 2^-24 each: a score is off by d = (3 * 2^-22 +
    3 hd 2^-24) scale sum |q k|, and by 2^-23 of its size from its scaling and M. A weight is off by
    2 ln 2^.. (d + that) + 2^-22, numerator and denominator alike, and the second product adds 3 * 2^-22
    and its own sums, 3 * 2^-24 a key."""
    hd = q.shape[1] // hq
    out = np.zeros((q.shape[0], hq, hd))
    tol = np.zeros_like(out)
    a = b = 0
    for n, m in zip(q_lens, k_lens):
        mask = seen(n, m, causal, window)
        some = mask.any(1)
        for h in range(hq):
            hk = h // (hq // hkv)
            x = q[a:a + n, h * hd:(h + 1) * hd].astype(np.float64)
            y = k[b:b + m, hk * hd:(hk + 1) * hd].astype(np.float64)
            z = v[b:b + m, hk * hd:(hk + 1) * hd].astype(np.float64)
            if not some.any():
                continue
            s = np.where(mask, scale * (x @ y.T), -np.inf)[some]
            size = np.where(mask, abs(scale) * (np.abs(x) @ np.abs(y).T), 0)[some].max(1, keepdims=True)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            out[a:a + n, h][some] = w @ z
            d = size * (3 * 2.0 ** -22 + (3 * hd + 2) * 2.0 ** -24)
            rel = 2 * d + 2 * 2.0 ** -22 + 3 * 2.0 ** -22 + 2 * 3 * m * 2.0 ** -24
            tol[a:a + n, h][some] = (w @ np.abs(z)) * rel
        a, b = a + n, b + m
    return out, tol


def check(got, want, tol, part=2.0 ** -17):
    """Every value within its bound, and the whole as near as independent roundings leave it: a
    score of about 10 is off by some 10 * 2^-22, a part of an operand that was left out by 2^-12."""
    got = got.reshape(want.shape).astype(np.float64)
    assert np.all(np.abs(got - want) <= tol + 1e-37), float((np.abs(got - want) - tol).max())
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= part * norm, float(np.linalg.norm(got - want) / norm)


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def rows(g, n, m, hq, hkv, hd):
    q = g.standard_normal((n, hq * hd)).astype(F)
    k = (g.standard_normal((m, hkv * hd)) * (1 + 3 * (g.random(hkv * hd) > 0.95))).astype(F)
    v = (g.standard_normal((m, hkv * hd)) * 0.5).astype(F)
    return q, k, v


LENS = [([1], None), ([64], None), ([65], None), ([63, 1, 128], None), ([0, 5, 0], None), ([200, 3, 0, 129, 40], None),
        ([700], None), ([3, 3, 3], [3, 100, 64]), ([17, 0, 130, 1], [400, 9, 131, 1]), ([40, 9], [20, 0]),
        (list(range(0, 40)), None), ([1, 1, 1, 1], [1, 700, 64, 65])]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd", [(2, 2, 64), (8, 1, 128), (5, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("case", range(len(LENS)))
def test_lengths_heads_and_masks(ctx, hq, hkv, hd, case):
    ql, kl = LENS[case]
    kl = ql if kl is None else kl
    print("[case] packed", hq, hkv, hd, ql, kl, flush=True)
    g = np.random.default_rng(case)
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(len(ql), sum(ql), max(sum(kl), 1), hq, hkv, hd)
    scale = hd ** -0.5
    for causal, window in ((False, 0), (True, 0), (True, 1), (True, 7), (True, 64), (True, 100), (True, 5000)):
        got = plan.attn(q, k, v, ql, kl, scale, causal, window)
        want, tol = attend(q, k, v, ql, kl, hq, hkv, scale, causal, window)
        check(got, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd,ql,kl,causal,window", [
    (2, 1, 128, [50], [9000], True, 0),  # few tiles: their keys over many workgroups
    (4, 4, 64, [129, 2], [5000, 4000], False, 0),
    (3, 3, 64, [2500, 31, 700], None, True, 0),
    (8, 2, 128, [1111], None, True, 300),
    (2, 2, 64, [300] * 20, [1500] * 20, False, 0),
    (16, 2, 128, [1] * 40 + [600], [900] * 40 + [800], True, 0),
    (1, 1, 128, [4100], None, True, 0),
    (4, 2, 64, [90, 400, 0, 513], None, True, 0),  # packed, with sequences of no rows and of few
    (8, 1, 128, [33, 385, 1, 64], None, True, 70),
    (2, 2, 64, [700, 3], [900, 5], True, 191), (2, 1, 64, [700, 3], [900, 5], True, 257), (4, 2, 128, [1000], None, True, 1),
    (1, 1, 128, [80, 600], [1600, 600], True, 130),  # long ones, each row of few keys
    (8, 8, 128, [200, 300, 250, 100, 33, 299, 128, 64, 1, 0, 257], None, True, 0),  # short ones, many tiles
    (4, 2, 64, [250] * 39 + [17], None, True, 90),
    (2, 1, 128, [40] * 300, None, True, 0)])  # short ones beyond two rounds of workgroups
def test_keys_split_over_workgroups(ctx, hq, hkv, hd, ql, kl, causal, window):
    print("[case] packed split", hq, hkv, hd, ql[:3], causal, window, flush=True)
    kl = ql if kl is None else kl
    g = np.random.default_rng(hq)
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(len(ql), sum(ql), sum(kl), hq, hkv, hd)
    got = plan.attn(q, k, v, ql, kl, hd ** -0.5, causal, window)
    check(got, *attend(q, k, v, ql, kl, hq, hkv, hd ** -0.5, causal, window))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd,ql,kl,causal,window", [
    (1024, 1, 64, [2, 0, 1], [70, 5, 9], True, 0), (1024, 1024, 64, [2, 1], [65, 1], False, 0),
    (512, 2, 128, [5], [66], True, 3), (1024, 4, 128, [1, 2], [900, 1], True, 0),
    (2, 2, 128, [1] * 1023 + [300], [3] * 1023 + [300], True, 0), (2, 1, 64, [0] * 1000 + [40] * 24, None, True, 0),
    (2, 1, 64, [1, 0] * 512, [0, 3] * 512, False, 0)])
def test_the_ends_of_the_ranges(ctx, hq, hkv, hd, ql, kl, causal, window):
    """As many heads and sequences as a plan takes."""
    print("[case] packed ends", hq, hkv, hd, len(ql), causal, window, flush=True)
    kl = ql if kl is None else kl
    g = np.random.default_rng(hq)
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(len(ql), sum(ql), sum(kl), hq, hkv, hd)
    got = plan.attn(q, k, v, ql, kl, hd ** -0.5, causal, window)
    check(got, *attend(q, k, v, ql, kl, hq, hkv, hd ** -0.5, causal, window))


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd,n,causal", [(2, 1, 128, 1500, True), (2, 2, 64, 2100, False), (16, 2, 64, 5000, True),
                                                (1, 1, 128, 9000, True), (20, 1, 64, 1, False)])
def test_the_same_bits_every_time(ctx, hq, hkv, hd, n, causal):
    """Whichever workgroup joins a tile's pieces."""
    print("[case] packed again", hq, hkv, hd, n, flush=True)
    g = np.random.default_rng(n)
    m = max(n, 3000)
    q, k, v = rows(g, n, m, hq, hkv, hd)
    plan = ctx.packed_attn(1, n, m, hq, hkv, hd)
    d_q, d_k, d_v, d_o = (_up(ctx, a) for a in (q, k, v, np.zeros_like(q)))
    qo, ko = _up(ctx, np.array([0, n], np.int32)), _up(ctx, np.array([0, m], np.int32))
    first = None
    for _ in range(25):
        d_o.upload(np.zeros_like(q))
        plan.attn_dev(1, n, m, n, m, qo, ko, d_q, d_k, d_v, hd ** -0.5, d_o, causal=causal)
        ctx.synchronize()
        got = d_o.download(F, q.size)
        assert first is None or np.array_equal(got, first)
        first = got


@pytest.mark.gpu
@pytest.mark.parametrize("n,stride", [(140, 1 << 23), (600, 1 << 21)])
def test_rows_far_apart(ctx, n, stride):
    """Rows of a projection more than 2^32 bytes apart, and of outputs."""
    print("[case] packed far", n, stride, flush=True)
    g = np.random.default_rng(n)
    hq, hkv, hd = 2, 1, 64
    q, k, v = rows(g, n, n, hq, hkv, hd)
    wide = hip.DeviceBuffer(ctx, ((n - 1) * stride + 4 * hd) * 4)
    x = np.concatenate([q, k, v], 1)
    at = lambda row, col=0: C.c_void_p(wide.ptr.value + (row * stride + col) * 4)  # noqa: E731
    for r in range(n):
        hip._check(hip.lib().vokra_hip_memcpy_htod(ctx._h, at(r), np.ascontiguousarray(x[r]).ctypes.data_as(C.c_void_p),
                                                   x[r].nbytes))
    d_q, d_k, d_v = (At(wide, c) for c in (0, 2 * hd, 3 * hd))
    d_o, d_small = _up(ctx, np.zeros_like(q)), [_up(ctx, a) for a in (q, k, v)]
    off = _up(ctx, np.array([0, n], np.int32))
    plan = ctx.packed_attn(1, n, n, hq, hkv, hd)
    want, tol = attend(q, k, v, [n], [n], hq, hkv, hd ** -0.5, True)
    plan.attn_dev(1, n, n, n, n, off, None, d_q, d_k, d_v, hd ** -0.5, d_o, causal=True, q_stride=stride, k_stride=stride,
                  v_stride=stride)
    ctx.synchronize()
    check(d_o.download(F, q.size), want, tol)
    few = _up(ctx, np.array([0, 3], np.int32))
    plan.attn_dev(1, 3, n, 3, n, few, off, d_small[0], d_k, d_v, hd ** -0.5, d_o, k_stride=stride, v_stride=stride)
    ctx.synchronize()
    check(d_o.download(F, 3 * hq * hd), *attend(q[:3], k, v, [3], [n], hq, hkv, hd ** -0.5))
    plan.attn_dev(1, n, n, n, n, off, None, *d_small, hd ** -0.5, wide, causal=True, out_stride=stride)
    ctx.synchronize()
    got = np.empty((n, hq * hd), F)
    for r in range(n):
        hip._check(hip.lib().vokra_hip_memcpy_dtoh(ctx._h, got[r].ctypes.data_as(C.c_void_p), at(r), got[r].nbytes))
    check(got, want, tol)


FEW = [(1, 1, 64, [1], [1]), (8, 1, 128, [1, 1, 1], [3, 900, 64]), (20, 20, 64, [5] * 6, [97, 1, 1500, 0, 16, 333]),
       (2, 2, 128, [7, 0, 16, 3], [40, 9, 2000, 17]), (6, 2, 64, [10, 1], [5000, 15]), (32, 1, 64, [1], [70]),
       (4, 2, 128, [16, 2], [33, 3000]), (16, 1, 128, [1], [20000]), (3, 3, 64, [32, 1], [9001, 70]),
       (4, 1, 128, [4, 8, 2], [700, 3, 1]), (2, 1, 64, [9, 0, 5], [4, 0, 300])]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(FEW)))
def test_few_rows(ctx, case):
    """Tokens, and candidates against their utterance."""
    hq, hkv, hd, ql, kl = FEW[case]
    print("[case] packed few", *FEW[case], flush=True)
    g = np.random.default_rng(case)
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(len(ql), sum(ql), sum(kl), hq, hkv, hd)
    for causal, window in ((False, 0), (True, 0), (True, 5)):
        got = plan.attn(q, k, v, ql, kl, hd ** -0.5, causal, window)
        check(got, *attend(q, k, v, ql, kl, hq, hkv, hd ** -0.5, causal, window))


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,causal", [([150, 70], [150, 70], True), ([3, 4], [150, 70], False)])
def test_values_of_any_size(ctx, ql, kl, causal):
    """Small and large operands, tiles of very different V, and scales of both signs and zero."""
    print("[case] packed sizes", ql, flush=True)
    g = np.random.default_rng(7)
    hq, hkv, hd = 4, 2, 64
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(2, sum(ql), sum(kl), hq, hkv, hd)
    tiles = np.repeat(10.0 ** g.integers(-30, 30, -(-sum(kl) // 64)), 64)[:sum(kl), None]
    with np.errstate(all="ignore"):
        for fq, fk, fv, scale in ((1e-20, 1e20, 1.0, 0.125), (1e18, 1e-18, 1e-30, 0.125), (1.0, 1.0, 1e36, 0.125),
                                  (1.0, 1.0, tiles, 0.125), (1e4, 1e4, 1.0, 1e-9), (1.0, 1.0, 1.0, -0.125),
                                  (1.0, 1.0, 1.0, 0.0), (30.0, 1.0, 1.0, 0.125), (1e-38, 1e-38, 1.0, 0.125),
                                  (1.0, 0.0, 1.0, 0.125), (0.0, 1.0, 0.0, 0.125)):
            x, y, z = (q * F(fq)).astype(F), (k * F(fk)).astype(F), (v * fv).astype(F)
            got = plan.attn(x, y, z, ql, kl, scale, causal)
            want, tol = attend(x, y, z, ql, kl, hq, hkv, float(F(scale)), causal)
            part = 2.0 ** -13 if fq == 30.0 else 2.0 ** -17  # (scores of some 300)
            if np.linalg.norm(want) > 0:
                check(got / np.abs(want).max(), want / np.abs(want).max(), tol / np.abs(want).max(), part)
            else:
                assert np.all(got == 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,hd,ql,kl,causal,window", [
    (2, 1, 64, [100, 90], [100, 90], True, 0), (2, 2, 128, [100, 90], [100, 90], True, 20),
    (3, 1, 64, [5, 4], [100, 90], True, 0), (2, 1, 64, [5, 4], [100, 90], False, 0), (2, 2, 128, [1, 1], [100, 90], True, 30),
    (2, 1, 64, [5, 4], [100, 90], True, 20), (2, 2, 128, [7, 13], [100, 90], True, 9), (4, 1, 64, [8, 6], [100, 90], True, 70),
    (2, 1, 128, [16, 9], [100, 90], True, 0), (2, 1, 64, [600, 90], [600, 90], True, 0), (2, 2, 128, [600, 90], [600, 90], True, 99),
    (64, 64, 128, [100, 90], [100, 90], True, 0), (160, 160, 64, [100, 90], [100, 90], True, 33)])  # in each way
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(ctx, hq, hkv, hd, ql, kl, causal, window):
    print("[case] packed nan", hq, hkv, hd, ql, causal, window, flush=True)
    g = np.random.default_rng(9)
    q, k, v = rows(g, sum(ql), sum(kl), hq, hkv, hd)
    plan = ctx.packed_attn(2, sum(ql), sum(kl), hq, hkv, hd)
    scale = hd ** -0.5
    want, tol = attend(q, k, v, ql, kl, hq, hkv, scale, causal, window)
    masks = [seen(n, m, causal, window) for n, m in zip(ql, kl)]
    for key in (0, 50, 80, 99):  # of the first sequence
        sees = np.concatenate([masks[0][:, key], np.zeros(ql[1], bool)])
        for bad in (np.nan, np.inf, -np.inf):
            y = k.copy()
            y[key, 3] = bad
            got = plan.attn(q, y, v, ql, kl, scale, causal, window).reshape(want.shape)
            hit = np.zeros(want.shape[:2], bool)
            hit[:, :hq // hkv] = sees[:, None]  # heads that read kv head 0
            assert np.all(np.isnan(got[hit]))
            assert np.all(np.abs(got[~hit] - want[~hit]) <= tol[~hit])
            z = v.copy()
            z[key, 3] = bad
            got = plan.attn(q, k, z, ql, kl, scale, causal, window).reshape(want.shape)
            at = np.zeros(want.shape, bool)
            at[:, :hq // hkv, 3] = sees[:, None]
            assert not np.any(np.isfinite(got[at]))
            assert np.all(np.abs(got[~at] - want[~at]) <= tol[~at])
    x = q.copy()
    x[1, 5] = np.nan
    got = plan.attn(x, k, v, ql, kl, scale, causal, window).reshape(want.shape)
    rest = np.ones(want.shape, bool)
    if np.concatenate([m.any(1) for m in masks])[1]:
        assert np.all(np.isnan(got[1, 0]))
        rest[1, 0] = False
    assert np.all(np.abs(got[rest] - want[rest]) <= tol[rest])


def _up(ctx, a):
    return hip.DeviceBuffer.from_array(ctx, a)


class At:
    def __init__(self, buf, at):
        self.ptr, self.keep = C.c_void_p(buf.ptr.value + 4 * at), buf


@pytest.mark.gpu
@pytest.mark.parametrize("ql,causal", [([30, 0, 101, 7], True), ([2, 0, 3, 1], False)])
def test_parts_of_a_projection_and_rows_that_no_sequence_has(ctx, ql, causal):
    """q, k and v in one buffer's rows; rows before the first and behind the last sequence hold NaN and
    are neither read into others nor written."""
    print("[case] packed strides", ql, flush=True)
    g = np.random.default_rng(4)
    hq, hkv, hd, before, behind = 4, 2, 64, 3, 9
    n = sum(ql) + before + behind
    w = (hq + 2 * hkv) * hd + 8
    x = g.standard_normal((n, w)).astype(F)
    x[:before] = x[n - behind:] = np.nan
    x[:, (hq + 2 * hkv) * hd:] = np.nan
    off = (before + np.concatenate([[0], np.cumsum(ql)])).astype(np.int32)
    plan = ctx.packed_attn(8, n + 5, n + 5, hq, hkv, hd)
    d_x, d_off = _up(ctx, x), _up(ctx, off)
    so = hq * hd + 4
    d_o = _up(ctx, np.full((n, so), 5.0, F))
    plan.attn_dev(len(ql), n, n, max(ql), max(ql), d_off, None, d_x, At(d_x, hq * hd), At(d_x, (hq + hkv) * hd), 0.125,
                  d_o, causal, 0, w, w, w, so)
    ctx.synchronize()
    got = d_o.download(F, n * so).reshape(n, so)
    assert np.all(got[:before] == 5.0) and np.all(got[n - behind:] == 5.0) and np.all(got[:, hq * hd:] == 5.0)
    r = x[before:n - behind]
    q, k, v = (np.ascontiguousarray(r[:, a * hd:b * hd]) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    check(got[before:n - behind, :hq * hd], *attend(q, k, v, ql, ql, hq, hkv, 0.125, causal))
    assert np.array_equal(d_x.download(F, x.size).reshape(x.shape), x, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("few", [False, True])
def test_offsets_out_of_order_or_range_are_passed_over(ctx, few):
    print("[case] packed offsets", few, flush=True)
    g = np.random.default_rng(5)
    hq, hkv, hd, n = 2, 1, 64, 200
    q, k, v = rows(g, n, n, hq, hkv, hd)
    plan = ctx.packed_attn(6, n, n, hq, hkv, hd)
    d_q, d_k, d_v, d_o = (_up(ctx, a) for a in (q, k, v, np.zeros((n, hq * hd), F)))
    most = 8 if few else 80
    good = np.array([0, 5, 13, 13, 20] if few else [0, 60, 140, 140, 200], np.int32)
    d_off, d_koff = _up(ctx, good), _up(ctx, good)

    def run(off, koff, done, max_q=most, max_k=most):
        d_off.upload(np.asarray(off, np.int32))
        d_koff.upload(np.asarray(koff, np.int32))
        d_o.upload(np.full((n, hq * hd), 7.0, F))
        plan.attn_dev(4, n, n, max_q, max_k, d_off, d_koff, d_q, d_k, d_v, 0.125, d_o, not few)
        ctx.synchronize()
        got = d_o.download(F, n * hq * hd).reshape(n, -1)
        ql, kl = np.diff(good)[:done], np.diff(good)[:done]
        m = int(ql.sum())
        check(got[:m], *attend(q[:m], k[:m], v[:m], ql, kl, hq, hkv, 0.125, not few))
        assert np.all(got[m:] == 7.0)
    run(good, good, 4)
    for i in (1, 2, 3, 4):
        for value in (-1, n + 1, 2 ** 31 - 1, -2 ** 31, good[i - 1] - 1 if i > 1 else -5):
            off = good.copy()
            off[i] = value
            run(off, good, i - 1)
            run(good, off, i - 1)
    run(good, good, 1, max_q=7 if few else 79)  # the second is longer than the bound
    run(good, good, 1, max_k=7 if few else 79)


@pytest.mark.gpu
@pytest.mark.parametrize("few", [False, True])
def test_in_a_graph_with_other_lengths(ctx, few):
    """One captured call serves other lengths within its bounds; two graphs share a plan."""
    print("[case] packed graph", few, flush=True)
    g = np.random.default_rng(6)
    hq, hkv, hd, n = 4, 1, 64, 400
    most = 8 if few else 300
    plan = ctx.packed_attn(5, n, n, hq, hkv, hd)
    d_q, d_k, d_v = (_up(ctx, np.zeros((n, h * hd), F)) for h in (hq, hkv, hkv))
    d_o = [_up(ctx, np.zeros((n, hq * hd), F)) for _ in (0, 1)]
    d_off, d_koff = _up(ctx, np.zeros(6, np.int32)), _up(ctx, np.zeros(6, np.int32))
    graphs = [ctx.capture(lambda o=o, c=c: plan.attn_dev(5, n, n, most, 300, d_off, d_koff, d_q, d_k, d_v, 0.125, o, c))
              for o, c in zip(d_o, (False, not few))]
    for ql, kl in (([3, 8, 0, 1, 5], [300, 20, 1, 0, 64]), ([8, 8, 8, 8, 8], [70] * 5),
                   ([1, 0, 0, 0, 0], [1, 0, 0, 0, 0]), ([2, 2, 2, 2, 2], [65, 64, 63, 1, 100])):
        if not few:
            ql = [x * 30 for x in ql] if max(ql) * 30 <= 240 and sum(ql) * 30 <= n else ql
        q, k, v = rows(g, n, n, hq, hkv, hd)
        for d, a in ((d_q, q), (d_k, k), (d_v, v)):
            d.upload(a)
        for d, x in ((d_off, ql), (d_koff, kl)):
            d.upload(np.concatenate([[0], np.cumsum(x)]).astype(np.int32))
        for _ in range(2):
            for graph in graphs:
                graph.launch()
        ctx.synchronize()
        a, b = sum(ql), sum(kl)
        for o, c in zip(d_o, (False, not few)):
            got = o.download(F, n * hq * hd).reshape(n, -1)[:a]
            check(got, *attend(q[:a], k[:b], v[:b], ql, kl, hq, hkv, 0.125, c))


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] packed refusals", flush=True)
    for a in ((0, 1, 1, 1, 1, 64), (1, 0, 1, 1, 1, 64), (1, 1, 0, 1, 1, 64), (1025, 1, 1, 1, 1, 64), (1, 2 ** 20 + 1, 1, 1, 1, 64),
              (1, 1, 2 ** 20 + 1, 1, 1, 64), (1, 1, 1, 3, 2, 64), (1, 1, 1, 0, 1, 64), (1, 1, 1, 1, 0, 64), (1, 1, 1, 1025, 1, 64)):
        with pytest.raises(hip.InvalidArgument):
            ctx.packed_attn(*a)
    with pytest.raises(hip.UnsupportedOp):
        ctx.packed_attn(1, 1, 1, 1, 1, 96)
    plan = ctx.packed_attn(2, 16, 16, 2, 1, 64)
    q, k, v, o = (hip.DeviceBuffer(ctx, 16 * 128 * 4) for _ in range(4))
    off = _up(ctx, np.array([0, 8, 16], np.int32))

    def bad(*a, **kw):
        with pytest.raises(hip.InvalidArgument):
            plan.attn_dev(*a, **kw)
    ok = (2, 16, 16, 8, 8, off, None, q, k, v, 0.125, o)
    plan.attn_dev(*ok)
    bad(3, *ok[1:])
    bad(2, 17, *ok[2:])
    bad(2, 16, 17, *ok[3:])
    bad(*ok[:10], float("nan"), o)
    bad(*ok[:10], float("inf"), o)
    bad(*ok, window=3)
    bad(*ok, q_stride=124)
    bad(*ok, q_stride=130)
    bad(*ok, k_stride=60)
    bad(*ok, v_stride=2 ** 23 + 4)
    bad(*ok, out_stride=127)
    bad(*ok[:7], At(q, 1), *ok[8:])
    bad(*ok[:8], At(k, 2), *ok[9:])
    bad(*ok[:9], At(v, 3), *ok[10:])
    bad(*ok[:11], At(o, 1))
    bad(*ok[:11], q)
    bad(*ok[:11], k)
    bad(*ok[:11], At(v, 16))
    bad(*ok[:11], off)
    null = type("At", (), {"ptr": None})
    for i in (5, 7, 8, 9, 11):
        bad(*ok[:i], null, *ok[i + 1:])
    plan.attn_dev(0, *ok[1:])
    plan.attn_dev(2, 0, *ok[2:])
    with pytest.raises(hip.InvalidArgument):
        plan.attn(np.zeros((4, 128)), np.zeros((4, 64)), np.zeros((4, 64)), [4, -1], [4, 0])
    with pytest.raises(hip.InvalidArgument):
        plan.attn(np.zeros((4, 128)), np.zeros((4, 64)), np.zeros((4, 64)), [3])
    with pytest.raises(hip.InvalidArgument):
        plan.attn(np.zeros((4, 128)), np.zeros((4, 64)), np.zeros((4, 64)), [4], [2, 2])
    assert plan.attn(np.zeros((0, 128)), np.zeros((0, 64)), np.zeros((0, 64)), []).shape == (0, 128)
    ctx.synchronize()


def test_missing_arguments_are_refused_without_a_device():
    L, null = hip.lib(), C.c_void_p()
    assert L.vokra_hip_packed_attn_create(null, 1, 1, 1, 1, 1, 64, C.byref(C.c_void_p())) == 5
    assert L.vokra_hip_packed_attn_dev(null, null, 1, 1, 1, 1, 1, null, null, null, 1, null, 1, null, 1, 1.0, 0, 0, null,
                                       1) == 5
    assert L.vokra_hip_packed_attn(null, null, 1, None, None, None, None, None, 1.0, 0, 0, None) == 5
    L.vokra_hip_packed_attn_destroy(None)
