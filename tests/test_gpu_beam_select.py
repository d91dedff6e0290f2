"""GPU parity of beam search's selection with the definition in extended precision."""
import ctypes as C

import numpy as np
import pytest

from vokra_amd import hip

F, LD = np.float32, np.longdouble


def select(x, scores, n_out, ended=None, end_token=-1):
    """The definition of the header; x [groups, beams, vocab]."""
    g, b, v = x.shape
    out = [np.full((g, n_out), -np.inf, F), np.full((g, n_out), -1, np.int32), np.full((g, n_out), -1, np.int32),
           np.ones((g, n_out), np.int32)]
    for i in range(g):
        rows = []  # (-total, beam, -logit, token)
        for j in range(b):
            s = scores[i, j]
            if not s > -np.inf:
                continue
            if ended is not None and ended[i, j]:
                rows.append(np.array([[-LD(s), j, 0, end_token]], LD))
                continue
            y = np.where(np.isnan(x[i, j]), -np.inf, x[i, j]).astype(LD)
            if y.max() in (np.inf, -np.inf):
                continue
            lse = y.max() + np.log(np.exp(y - y.max()).sum())
            # totals in 64 bits decide, as they do on the device
            total = (LD(s) + (y - lse)).astype(np.float64)
            at = np.flatnonzero(y > -np.inf)
            if at.size > 4 * n_out:  # (logits at the border all stay)
                at = at[y[at] >= np.partition(y[at], -n_out)[-n_out]]
            rows.append(np.stack([-total[at].astype(LD), np.full(at.size, j, LD), -y[at], at.astype(LD)], 1))
        if not rows:
            continue
        rows = np.concatenate(rows)
        first = rows[np.lexsort(rows.T[::-1])][:n_out]
        m = len(first)
        out[0][i, :m] = (-first[:, 0]).astype(F)
        out[1][i, :m], out[2][i, :m] = first[:, 1].astype(int), first[:, 3].astype(int)
        over = first[:, 3].astype(int) == end_token
        if ended is not None:
            over |= ended[i][first[:, 1].astype(int)].astype(bool)
        out[3][i, :m] = over
    return out


def check(got, want, gap=True):
    for a, b in zip(got[1:], want[1:]):
        assert np.array_equal(a, b)
    # a total's f32 rounding is half a step; the sum of exponentials is f32 work: an argument below
    # 2^7 in size rounded three times, the exponential's unit, 32 adds, each 2^-24 of it at most: under
    # (3 * 2^7 + 1 + 32) * 2^-24 = 2.5e-5 of the sum if all fell one way, which ln carries over as it is
    a, b = got[0].astype(np.float64), want[0].astype(np.float64)
    ok = np.isfinite(b)
    assert np.array_equal(np.isfinite(a), ok)
    assert np.all(np.abs(a[ok] - b[ok]) <= 2.5e-5 + np.abs(b[ok]) * 2.0 ** -23)


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def logits(g, *shape):
    """Rows whose best tokens lie apart (multiples of 2^-10 of the row's own order): totals of
    different beams are then apart by more than the sums' rounding, or equal."""
    return np.round(g.standard_normal(shape) * 3000).astype(F) / F(1024)


@pytest.mark.gpu
@pytest.mark.parametrize("groups,beams,vocab,n_out", [
    (1, 1, 1, 1), (2, 3, 2, 5), (1, 5, 33, 10), (3, 2, 1000, 4), (2, 4, 4096, 8), (1, 5, 4097, 64), (2, 32, 515, 64),
    (1, 5, 51865, 10), (7, 5, 51866, 5), (2, 12, 130001, 24), (9, 8, 51866, 16), (1, 1, 300000, 64), (1, 2, 600001, 3),
    (65, 1, 8191, 1)])
def test_the_best_of_groups(ctx, groups, beams, vocab, n_out):
    print("[case] beam", groups, beams, vocab, n_out, flush=True)
    g = np.random.default_rng(vocab)
    plan = ctx.beam_select(groups, beams, vocab, n_out)
    x = logits(g, groups, beams, vocab)
    scores = -g.random((groups, beams)).astype(F) * 5
    check(plan.select(x, scores, n_out), select(x, scores, n_out))
    ended = (g.random((groups, beams)) < 0.4).astype(np.int32)
    end = int(g.integers(0, vocab))
    x[g.random(x.shape) < 0.5] = -np.inf
    check(plan.select(x, scores, n_out, ended, end), select(x, scores, n_out, ended, end))
    scores[:, 1:] = -np.inf  # a first step: one beam of each group
    check(plan.select(x, scores, n_out, None, end), select(x, scores, n_out, None, end))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,beams", [(9000, 4), (600000, 2), (300000, 3)])
def test_ties_go_to_the_lower_beam_and_token(ctx, vocab, beams):
    """Constant rows (every column ties), a few values only, zeros of both signs, equal beams."""
    print("[case] beam ties", vocab, flush=True)
    g = np.random.default_rng(1)
    x = np.zeros((4, beams, vocab), F)
    x[0] = -3.0
    x[1] = g.integers(0, 2, (beams, vocab))
    x[2] = np.where(g.random((beams, vocab)) < 0.5, 0.0, -0.0)
    x[2, :, 4090:4100] = 1.0
    x[3] = x[1, 0]  # equal rows: where they start in memory does not matter
    x[3, :, 4096:8191] = 2.0
    scores = np.zeros((4, beams), F)
    for n_out in (1, 7, 33, 64):
        plan = ctx.beam_select(4, beams, vocab, n_out)
        got = plan.select(x, scores, n_out)
        assert np.array_equal(got[1][[0, 3]], np.zeros((2, n_out)))
        assert np.array_equal(got[2][0], np.arange(n_out))
        # rows of different sums may be next to each other: those of equal rows are what is compared
        want = select(x, scores, n_out)
        for a, b in zip(got[1:3], want[1:3]):
            assert np.array_equal(a[[0, 3]], b[[0, 3]])
        for i in (1, 2):
            for j in range(beams):
                mine = got[2][i][got[1][i] == j]
                falling = np.argsort(-x[i, j], kind="stable")
                assert np.array_equal(mine, falling[:mine.size])


@pytest.mark.gpu
def test_rows_where_nothing_is_left_and_values_that_are_not_finite(ctx):
    print("[case] beam edges", flush=True)
    g = np.random.default_rng(2)
    x = logits(g, 7, 2, 5000)
    x[0] = -np.inf  # no token
    x[1, 0] = np.nan
    x[2, 0, 17] = np.inf  # no continuation of that beam
    x[3, :, 100:] = np.nan
    x[4] = -3.4e38
    x[5, 0] = 3.4e38
    x[6, 0, 1:], x[6, 1, :] = -np.inf, -np.inf  # one token in all
    scores = np.zeros((7, 2), F) - [[0.0, 0.25]]
    scores = scores.astype(F)
    ended = np.zeros((7, 2), np.int32)
    plan = ctx.beam_select(7, 2, 5000, 12)
    with np.errstate(all="ignore"):
        check(plan.select(x, scores, 12, ended, 3), select(x, scores, 12, ended, 3))
        ended[6] = [0, 1]
        ended[0] = [7, -1]  # any value but 0
        scores[4] = [np.nan, -np.inf]
        scores[5, 1] = -1e30
        check(plan.select(x, scores, 12, ended, 3), select(x, scores, 12, ended, 3))
    got = plan.select(x[:0], scores[:0], 12)
    assert all(a.shape == (0, 12) for a in got)


def _up(ctx, a):
    return hip.DeviceBuffer.from_array(ctx, a)


@pytest.mark.gpu
def test_strides_in_place_and_in_a_graph(ctx):
    """Steps that feed each other on the device: scores and ended in place, four replays."""
    print("[case] beam steps", flush=True)
    g = np.random.default_rng(3)
    groups, beams, vocab, stride, end = 3, 4, 777, 1001, 5
    plan = ctx.beam_select(4, 5, 1000, 9)
    scores = np.full((groups, beams), -np.inf, F)
    scores[:, 0] = 0.0
    ended = np.zeros((groups, beams), np.int32)
    d_x = _up(ctx, np.zeros(groups * beams * stride + 1, F))
    at = type("At", (), {"ptr": C.c_void_p(d_x.ptr.value + 4)})  # rows on no 16-byte boundary
    d_s, d_e = _up(ctx, scores), _up(ctx, ended)
    d_p, d_t = (_up(ctx, np.zeros((groups, beams), np.int32)) for _ in (0, 1))
    graph = None
    for step in range(5):
        x = np.full((groups * beams, stride), 99.0, F)
        x[:, :vocab] = logits(g, groups * beams, vocab)
        x[:, end] += 4.0
        d_x.upload(np.concatenate([[0.0], x.reshape(-1)]).astype(F))
        want = select(x[:, :vocab].reshape(groups, beams, vocab), scores, beams, ended, end)
        run = lambda: plan.select_dev(groups, beams, vocab, beams, at, d_s, d_s, d_p, d_t, d_e, end, d_e, stride)  # noqa: E731
        if graph is None:
            graph = ctx.capture(run)
        graph.launch()
        ctx.synchronize()
        got = [d_s.download(F, groups * beams)] + [d.download(np.int32, groups * beams) for d in (d_p, d_t, d_e)]
        got = [a.reshape(groups, beams) for a in got]
        check(got, want)
        scores, ended = got[0], got[3]


@pytest.mark.gpu
def test_rows_far_apart(ctx):
    """Rows of logits more than 2^32 bytes apart."""
    print("[case] beam far", flush=True)
    g = np.random.default_rng(4)
    x, stride = logits(g, 1, 2, 5000), (1 << 30) + 3
    wide = hip.DeviceBuffer(ctx, (stride + 5000) * 4)
    for b in (0, 1):
        hip._check(hip.lib().vokra_hip_memcpy_htod(ctx._h, C.c_void_p(wide.ptr.value + b * stride * 4),
                                                   x[0, b].ctypes.data_as(C.c_void_p), x[0, b].nbytes))
    scores = np.array([[-1.0, -2.0]], F)
    d_s = hip.DeviceBuffer.from_array(ctx, scores)
    out = [hip.DeviceBuffer.from_array(ctx, np.zeros((1, 7), t)) for t in (F, np.int32, np.int32, np.int32)]
    ctx.beam_select(1, 2, 5000, 7).select_dev(1, 2, 5000, 7, wide, d_s, *out[:3], d_out_ended=out[3], stride=stride)
    ctx.synchronize()
    got = [b.download(t, 7).reshape(1, 7) for b, t in zip(out, (F, np.int32, np.int32, np.int32))]
    check(got, select(x, scores, 7))


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] beam refusals", flush=True)
    for a in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 33, 1, 1), (1, 1, 2 ** 24 + 1, 1), (1, 1, 1, 65), (1, 1, 0, 1), (1, 1, 1, 0),
              (65536, 1, 1, 1), (30000, 3, 1, 1)):
        with pytest.raises(hip.InvalidArgument):
            ctx.beam_select(*a)
    plan = ctx.beam_select(2, 4, 100, 8)
    x, s, e = (hip.DeviceBuffer(ctx, 4096) for _ in range(3))
    o = [hip.DeviceBuffer(ctx, 256) for _ in range(4)]

    def bad(*a, **kw):
        with pytest.raises(hip.InvalidArgument):
            plan.select_dev(*a, **kw)
    bad(3, 4, 100, 4, x, s, *o[:3])
    bad(2, 5, 100, 4, x, s, *o[:3])
    bad(2, 4, 101, 4, x, s, *o[:3])
    bad(2, 4, 100, 9, x, s, *o[:3])
    bad(2, 4, 100, 0, x, s, *o[:3])
    bad(2, 4, 100, 4, x, s, *o[:3], stride=99)
    bad(2, 4, 100, 4, x, s, *o[:3], d_ended=e)  # no end token
    bad(2, 4, 100, 4, x, s, *o[:3], d_ended=e, end_token=100)
    bad(2, 4, 100, 4, x, s, *o[:3], end_token=-2)
    bad(2, 4, 100, 4, x, s, o[0], o[1], o[1])
    bad(2, 4, 100, 4, x, s, x, o[1], o[2])
    bad(2, 4, 100, 8, x, s, s, o[1], o[2])  # in place, but not of the same size
    bad(2, 4, 100, 4, x, s, o[0], s, o[2])
    bad(2, 4, 100, 4, x, s, *o[:3], d_ended=e, end_token=1, d_out_ended=s)
    part = type("At", (), {"ptr": C.c_void_p(s.ptr.value + 4)})
    bad(2, 4, 100, 4, x, s, part, o[1], o[2])
    plan.select_dev(0, 4, 100, 4, x, s, *o[:3])
    with pytest.raises(hip.InvalidArgument):
        plan.select(np.zeros((2, 4, 100)), np.zeros((2, 3)), 4)
    with pytest.raises(hip.InvalidArgument):
        plan.select(np.zeros((2, 4, 100)), np.zeros((2, 4)), 4, np.zeros(8), 3)
    ctx.synchronize()


def test_missing_arguments_are_refused_without_a_device():
    L, null = hip.lib(), C.c_void_p()
    assert L.vokra_hip_beam_create(null, 1, 1, 1, 1, C.byref(C.c_void_p())) == 5
    assert L.vokra_hip_beam_select_dev(null, null, 1, 1, 1, 1, 1, *[null] * 3, -1, *[null] * 4) == 5
    assert L.vokra_hip_beam_select(null, null, 1, 1, 1, 1, None, None, None, -1, None, None, None, None) == 5
    L.vokra_hip_beam_destroy(None)


def test_the_model_of_the_selection():
    """By hand: two beams, the second 0.5 behind, one of them ended."""
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.9, 0.05, 0.05]]], F))
    s, p, t, e = select(x, np.array([[0.0, -0.5]], F), 3)
    assert p.tolist() == [[1, 0, 0]] and t.tolist() == [[0, 0, 1]] and e.tolist() == [[0, 0, 0]]
    assert np.allclose(s, [[np.log(0.9) - 0.5, np.log(0.5), np.log(0.25)]])
    s, p, t, e = select(x, np.array([[0.0, -0.5]], F), 5, np.array([[0, 1]]), 2)
    assert p.tolist() == [[1, 0, 0, 0, -1]] and t.tolist() == [[2, 0, 1, 2, -1]] and e.tolist() == [[1, 0, 0, 1, 1]]
