"""GPU parity of the logits rules: the same f32 operations in numpy, bit for bit."""
import ctypes as C

import numpy as np
import pytest

from vokra_amd import hip

F = np.float32


def rules(x, history=None, repetition=None, presence=None, frequency=None, biases=None, mask=None):
    """The rules of the header, one row at a time, every operation in f32."""
    x = np.array(x, F)
    rows, vocab = x.shape
    nxt = np.full(rows, -1, np.int32)
    for r in range(rows):
        y = x[r]
        if history is not None:
            ids = np.asarray(history[r], np.int64)
            n = np.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab)
            h = n > 0
            rep = F(1) if repetition is None else F(repetition[r])
            pres = F(0) if presence is None else F(presence[r])
            freq = F(0) if frequency is None else F(frequency[r])
            with np.errstate(all="ignore"):
                y[h] = np.where(y[h] > 0, y[h] / rep, y[h] * rep)
                y[h] = y[h] - (pres + freq * n[h].astype(F))
        for i, b in ({i: b for i, b in biases[r]} if biases is not None else {}).items():
            if 0 <= i < vocab:
                y[i] = y[i] + F(b)
        if mask is not None:
            y[~(mask if mask.ndim == 1 else mask[r])] = -np.inf
        z = np.where(np.isnan(y), -np.inf, y)
        if z.max() > -np.inf:
            nxt[r] = int(np.argmax(z))
    return x, nxt


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def same(got, want):
    assert np.array_equal(got[0], want[0], equal_nan=True)
    assert np.array_equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 32), (2, 33), (5, 1000), (1, 4096), (2, 4097), (7, 51866),
                                        (33, 8191), (2, 130001), (41, 51866)])
def test_every_rule_at_once_and_alone(ctx, rows, vocab):
    print("[case] rules", rows, vocab, flush=True)
    g = np.random.default_rng(vocab)
    x = (g.standard_normal((rows, vocab)) * 3).astype(F)
    pool = g.integers(0, vocab, 50)
    kw = dict(history=[g.choice(pool, g.integers(0, 700)) for _ in range(rows)],
              repetition=g.uniform(1, 1.5, rows), presence=g.uniform(-1, 1, rows), frequency=g.uniform(0, 1, rows),
              biases=[[(int(i), float(b)) for i, b in zip(g.integers(0, vocab, n), g.normal(0, 5, n))]
                      for n in g.integers(0, 60, rows)], mask=g.random((rows, vocab)) < 0.3)
    same(ctx.logits_rules(x, **kw), rules(x, **kw))
    for names in (("history", "repetition"), ("history", "presence"), ("history", "frequency"), ("biases",), ("mask",), ()):
        one = {n: kw[n] for n in names}
        same(ctx.logits_rules(x, **one), rules(x, **one))
    one = dict(mask=kw["mask"][0])  # one mask for all rows
    same(ctx.logits_rules(x, **one), rules(x, **one))


@pytest.mark.gpu
def test_rows_where_nothing_is_left_ties_and_values_that_are_not_finite(ctx):
    print("[case] rules edges", flush=True)
    vocab = 9000
    x = np.full((9, vocab), -1.0, F)
    mask = np.ones((9, vocab), bool)
    mask[0] = False  # nothing is left
    x[1] = -np.inf
    x[2] = np.nan
    x[3, [70, 4500, 8999]] = 2.0  # a tie over workgroups: the lowest
    x[4, 8000] = np.inf
    x[5, 0], x[5, 1] = np.nan, -0.5
    mask[6] = False
    mask[6, 8999] = True
    x[7] = -3.4e38
    mask[8, :8999] = False
    x[8, 8999] = -np.inf
    kw = dict(mask=mask, history=[[4, 4, 8000]] * 9, repetition=[2.0] * 9, presence=[0.5] * 9, frequency=[1e38] * 9)
    for some in ({"mask": mask}, kw, {}):
        same(ctx.logits_rules(x, **some), rules(x, **some))
    assert rules(x, mask=mask)[1].tolist() == [-1, -1, -1, 70, 8000, 1, 8999, 0, -1]


@pytest.mark.gpu
def test_padding_ids_and_ids_given_twice(ctx):
    print("[case] rules ids", flush=True)
    x = np.random.default_rng(0).standard_normal((3, 5000)).astype(F)
    kw = dict(history=[[-1, -1, 7, 5000, 2 ** 31 - 1, 7], [], [-2 ** 31, 4999]], repetition=[1.3, 1.3, 0.7],
              biases=[[(7, 1.0), (7, -2.0), (7, 0.5)], [(-1, 9.0), (5000, 9.0)], [(4999, 1.0)] * 300 + [(4999, 4.0)]],
              frequency=[0.25, 0.0, 0.0])
    same(ctx.logits_rules(x, **kw), rules(x, **kw))


@pytest.mark.gpu
def test_a_long_history(ctx):
    print("[case] rules history", flush=True)
    g = np.random.default_rng(0)
    x = g.standard_normal((2, 20000)).astype(F)
    kw = dict(history=[g.integers(0, 20000, 300000), np.full(100000, 3)], frequency=[0.01, 0.001], presence=[0.1, 0])
    same(ctx.logits_rules(x, **kw), rules(x, **kw))


def _up(ctx, a):
    return hip.DeviceBuffer.from_array(ctx, a)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,stride,shift", [(5000, 5003, 0), (4999, 5000, 1), (51866, 51866, 0), (513, 515, 3)])
def test_strides_in_place_and_single_outputs(ctx, vocab, stride, shift):
    """Rows at any float offset: what lies between them stays; out in place, out
    alone, next alone."""
    print("[case] rules strides", vocab, stride, shift, flush=True)
    rows = 4
    g = np.random.default_rng(1)
    flat = g.standard_normal(rows * stride + 8).astype(F)
    x = np.lib.stride_tricks.as_strided(flat[shift:], (rows, vocab), (4 * stride, 4)).copy()
    hist = np.arange(0, 4000, 7, dtype=np.int32) % vocab
    off = np.array([0, 100, 100, hist.size, hist.size], np.int32)
    history = [hist[off[r]:off[r + 1]] for r in range(rows)]
    words = -(-vocab // 32)
    mask = g.integers(0, 2 ** 32, (rows, words + 2), dtype=np.uint64).astype(np.uint32)
    allowed = np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool)
    bufs = [_up(ctx, a) for a in (hist, off, np.full(rows, 1.25, F), mask)]
    ru = hip.LogitsRules(n_hist=hist.size, hist=bufs[0], hist_offsets=bufs[1], repetition=bufs[2], mask=bufs[3],
                         mask_stride=words + 2)
    want = rules(x, history=history, repetition=[1.25] * rows, mask=allowed)
    d, o = _up(ctx, flat), _up(ctx, np.full_like(flat, 5.0))
    at = lambda b: type("P", (), {"ptr": C.c_void_p(b.ptr.value + 4 * shift)})()  # noqa: E731
    nxt = [_up(ctx, np.full(rows, 77, np.int32)) for _ in range(3)]

    def rows_of(a):
        return np.lib.stride_tricks.as_strided(a[shift:], (rows, vocab), (4 * stride, 4))
    ctx.logits_rules_dev(rows, vocab, at(d), ru, None, nxt[0], stride=stride)
    ctx.logits_rules_dev(rows, vocab, at(d), ru, at(o), None, stride=stride)
    ctx.synchronize()
    got = o.download(F, flat.size)
    assert np.array_equal(d.download(F, flat.size), flat)
    assert np.array_equal(rows_of(got), want[0])
    between = np.full_like(flat, 5.0)
    rows_of(between)[:] = want[0]
    assert np.array_equal(got, between)
    ctx.logits_rules_dev(rows, vocab, at(d), ru, at(d), nxt[1], stride=stride)
    ctx.synchronize()
    rows_of(flat)[:] = want[0]
    assert np.array_equal(d.download(F, flat.size), flat)
    for n in nxt[:2]:
        assert np.array_equal(n.download(np.int32, rows), want[1])


@pytest.mark.gpu
def test_device_offsets_never_read_beyond_the_lists(ctx):
    print("[case] rules offsets", flush=True)
    x = np.random.default_rng(0).standard_normal((3, 100)).astype(F)
    ids = np.array([1, 2, 3, 4], np.int32)
    for off in ([0, 2, 90, 2 ** 31 - 1], [-5, 2, 1, 4], [3, 3, 3, -7]):
        bufs = [_up(ctx, a) for a in (ids, np.array(off, np.int32), np.full(3, 2, F), np.arange(4, dtype=F))]
        ru = hip.LogitsRules(n_hist=4, hist=bufs[0], hist_offsets=bufs[1], repetition=bufs[2], n_bias=4,
                             bias_ids=bufs[0], bias=bufs[3], bias_offsets=bufs[1])
        cut = [(max(a, 0), max(min(b, 4), max(a, 0))) for a, b in zip(off[:-1], off[1:])]
        kw = dict(history=[ids[a:b] for a, b in cut], repetition=[2] * 3,
                  biases=[[(int(i), float(i - 1)) for i in ids[a:b]] for a, b in cut])
        d, nxt = _up(ctx, x), _up(ctx, np.zeros(3, np.int32))
        ctx.logits_rules_dev(3, 100, d, ru, d, nxt)
        ctx.synchronize()
        same((d.download(F, 300).reshape(3, 100), nxt.download(np.int32, 3)), rules(x, **kw))


@pytest.mark.gpu
def test_more_rows_than_one_launch_takes(ctx):
    print("[case] rules many rows", flush=True)
    rows, vocab = 50000, 8193
    x = np.zeros((rows, vocab), F)
    g = np.random.default_rng(0)
    at = g.integers(0, vocab, rows).astype(np.int32)
    x[np.arange(rows), at] = 1.0
    d, nxt = _up(ctx, x), _up(ctx, np.zeros(rows, np.int32))
    off = _up(ctx, np.r_[np.arange(rows), rows].astype(np.int32))
    rep = _up(ctx, np.where(np.arange(rows) % 2, 0.5, 2.0).astype(F))
    pres = _up(ctx, np.where(np.arange(rows) % 3, 0.0, 3.0).astype(F))  # a third of the rows lose their largest
    ctx.logits_rules_dev(rows, vocab, d, hip.LogitsRules(n_hist=rows, hist=_up(ctx, at), hist_offsets=off,
                                                         repetition=rep, presence=pres), None, nxt)
    ctx.synchronize()
    want = np.where(np.arange(rows) % 3, at, np.where(at == 0, 1, 0))
    assert np.array_equal(nxt.download(np.int32, rows), want)


@pytest.mark.gpu
def test_a_captured_call_replays(ctx):
    print("[case] rules graph", flush=True)
    g = np.random.default_rng(0)
    rows, vocab = 3, 9001
    x = g.standard_normal((rows, vocab)).astype(F)
    d, o, nxt = _up(ctx, x), _up(ctx, x), _up(ctx, np.zeros(rows, np.int32))
    hist, off = _up(ctx, np.zeros(30, np.int32)), _up(ctx, np.array([0, 10, 20, 30], np.int32))
    rep = _up(ctx, np.full(rows, 1.5, F))
    ru = hip.LogitsRules(n_hist=30, hist=hist, hist_offsets=off, repetition=rep)
    ctx.logits_rules_dev(rows, vocab, d, ru, o, nxt)
    graph = ctx.capture(lambda: ctx.logits_rules_dev(rows, vocab, d, ru, o, nxt))
    for _ in range(4):
        h = g.integers(-1, vocab, 30).astype(np.int32)
        x = g.standard_normal((rows, vocab)).astype(F)
        hist.upload(h)
        d.upload(x)
        graph.launch()
        ctx.synchronize()
        got = o.download(F, x.size).reshape(x.shape), nxt.download(np.int32, rows)
        kw = dict(history=list(h.reshape(3, 10)), repetition=[1.5] * 3)
        same(got, rules(x, **kw))
        same(ctx.logits_rules(x, **kw), rules(x, **kw))  # eager work between the replays


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] rules refusals", flush=True)
    b = _up(ctx, np.zeros(4096, F))
    ru, null = hip.LogitsRules(), type("P", (), {"ptr": C.c_void_p()})()
    half = type("P", (), {"ptr": C.c_void_p(b.ptr.value + 64)})()
    for call in (lambda: ctx.logits_rules_dev(1, 0, b, ru, b, b), lambda: ctx.logits_rules_dev(1, (1 << 24) + 1, b, ru, b, b),
                 lambda: ctx.logits_rules_dev(65536, 10, b, ru, b, b), lambda: ctx.logits_rules_dev(1, 10, b, ru, b, b, stride=9),
                 lambda: ctx.logits_rules_dev(1, 10, null, ru, b, b), lambda: ctx.logits_rules_dev(1, 10, b, ru, None, None),
                 lambda: ctx.logits_rules_dev(2, 10, b, ru, half, None),
                 lambda: ctx.logits_rules_dev(1, 10, b, hip.LogitsRules(n_hist=3), b, b),
                 lambda: ctx.logits_rules_dev(1, 10, b, hip.LogitsRules(n_bias=3), b, b),
                 lambda: ctx.logits_rules_dev(1, 100, b, hip.LogitsRules(mask=b, mask_stride=3), b, b),
                 lambda: ctx.logits_rules(np.zeros((2, 10)), history=[[1]]),
                 lambda: ctx.logits_rules(np.zeros((2, 10)), presence=[1]),
                 lambda: ctx.logits_rules(np.zeros((2, 10)), mask=np.ones((3, 10)))):
        with pytest.raises(hip.InvalidArgument):
            call()
    x, out, off = np.zeros((2, 10), F), np.zeros((2, 10), F), np.array([0, 3, 2], np.int32)
    c = hip._LogitsRules()
    c.n_hist, c.hist, c.hist_offsets = 3, off.ctypes.data, off.ctypes.data
    args = (ctx._h, 2, 10, hip._ptr(x, C.c_float), C.byref(c), hip._ptr(out, C.c_float), None)
    assert hip.lib().vokra_hip_logits_rules(*args) == 5  # offsets out of order
    off[:] = [0, 1, 4]
    assert hip.lib().vokra_hip_logits_rules(*args) == 5  # beyond the list
    ctx.logits_rules_dev(0, 10, null, ru, None, None)


def test_missing_arguments_are_refused_without_a_device():
    L, null = hip.lib(), C.c_void_p()
    assert L.vokra_hip_logits_rules_dev(null, 1, 1, 1, null, None, null, null) == 5
    assert L.vokra_hip_logits_rules(null, 1, 1, None, None, None, None) == 5
