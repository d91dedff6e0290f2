"""GPU parity of the block-scaled KV cache with its numpy restatement
(tests/bkv_model.py): rounding and planning exactly, attention within the bound
that the restatement derives for an f32 evaluation."""
import numpy as np
import pytest

from tests import bkv_model as bm
from vokra_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


class _Ids:
    def __init__(self, ctx, a):
        self.b = hip.DeviceBuffer.from_array(ctx, np.ascontiguousarray(a, np.int32))
        self.ptr = self.b.ptr


class Pair:
    """The device cache and its restatement, driven together."""

    def __init__(self, ctx, n_layer, n_head, hd, n_seq, max_time, bs, n_page, max_rows, codec=0, seed=0):
        args = (n_layer, n_head, hd, n_seq, max_time, bs, n_page, max_rows, codec)
        self.ctx, self.dev, self.ref = ctx, ctx.block_kv_cache(*args), bm.Cache(*args)
        self.g = np.random.default_rng(seed)

    def rows(self, n):
        w = self.ref.n_head * self.ref.hd
        return [(self.g.standard_normal((n, w)) * np.exp(self.g.uniform(-2, 2, (n, 1)))).astype(np.float32)
                for _ in (0, 1)]

    def step(self, seqs, starts, counts, write=True):
        want, done = self.ref.step(list(seqs), list(starts), list(counts))
        assert self.outcome(lambda: self.dev.step(seqs, starts, counts)) == want
        if want:
            with pytest.raises(hip._ERRORS[want]):
                self.dev.status()
        else:
            assert self.dev.status() == done
        n = int(np.maximum(counts, 0).sum())
        if write:
            for layer in range(self.ref.n_layer):
                k, v = self.rows(n)
                self.dev.write(layer, k, v)
                self.ref.write(layer, k, v)
        return n

    @staticmethod
    def outcome(call):
        try:
            call()
            return bm.OK
        except (hip.InvalidArgument, hip.KvCacheExhausted) as e:
            return e.code

    def both(self, name, *args):
        want, _ = getattr(self.ref, name)(*args)
        assert self.outcome(lambda: getattr(self.dev, name)(*args)) == want

    def check_state(self):
        r = self.ref
        assert self.dev.pages() == (r.free_pages(), r.n_page - r.free_pages())
        for s in range(r.n_seq):
            assert self.dev.length(s) == r.len[s], s
            assert [self.dev.page_of(s, b) for b in range(len(r.table[s]) + 1)] == r.table[s] + [-1], s

    def check_rows(self):
        r = self.ref
        ids = [(s, t) for s in range(r.n_seq) for t in range(r.len[s])] + [(0, r.len[0]), (-1, 0), (r.n_seq, 0), (0, -1)]
        s, t = (np.array(x) for x in zip(*ids))
        for layer in range(r.n_layer):
            got = self.dev.read(layer, s, t)
            held = [r.held(layer, x) for x in range(r.n_seq)]
            for side in (0, 1):
                want = np.concatenate([h[side].reshape(-1, r.n_head * r.hd) for h in held] +
                                      [np.zeros((4, r.n_head * r.hd), np.float32)])
                assert np.array_equal(got[side], want, equal_nan=True), (layer, side)

    def check_attn(self, layer, n_rows, n_head_q, scale=None, q=None):
        r = self.ref
        scale = r.hd ** -0.5 if scale is None else scale
        if q is None:
            q = self.g.standard_normal((n_rows, n_head_q * r.hd)).astype(np.float32) * 2
        mark = np.full_like(q, 7.5)
        got = self.dev.attn(layer, q, n_head_q, scale, out=mark.copy())
        want, tol = r.attn(layer, q, n_head_q, np.float32(scale))
        out = np.isnan(tol) & np.isnan(want)
        done = sum(n for _, _, n, _ in r.plan)
        assert np.array_equal(got[done:], mark[done:])
        got, want, tol, out = got[:done], want[:done], tol[:done], out[:done]
        assert np.array_equal(np.isnan(got), out)
        err = np.abs(got.astype(np.float64) - want) / tol
        assert not np.any(err[~out] > 1), f"{np.nanmax(err)} of the bound"
        return got


@pytest.mark.parametrize("codec", [0, 1])
@pytest.mark.parametrize("bs,hd,heads", [(16, 64, 3), (32, 128, 1), (64, 64, 2), (16, 128, 2)])
def test_rows_are_held_as_the_definition_says_however_they_come(ctx, codec, bs, hd, heads):
    """The same rows in one step, token by token, and in ragged steps: bit-equal
    to the restatement, and to each other."""
    print("[case] bkv rows", codec, bs, hd, heads, flush=True)
    n = 3 * bs + 7
    p = Pair(ctx, 2, heads, hd, 3, n + 5, bs, 12, 3 * n, codec)
    whole = [p.rows(n) for _ in range(2)]
    cuts = [np.arange(n + 1), np.unique(np.r_[0, p.g.integers(1, n, 5), bs, n]), np.array([0, n])]
    for s, c in enumerate(cuts):
        for a, b in zip(c[:-1], c[1:]):
            assert p.ref.step([s], [a], [b - a])[0] == bm.OK
            p.dev.step([s], [a], [b - a])
            for layer in range(2):
                k, v = (x[a:b] for x in whole[layer])
                p.dev.write(layer, k, v)
                p.ref.write(layer, k, v)
    p.check_state()
    p.check_rows()


@pytest.mark.parametrize("codec", [0, 1])
def test_rounding_of_every_magnitude(ctx, codec):
    """Blocks from subnormal to the largest f32, zeros, ties, and values that are
    not finite (the block reads as NaN, its neighbours do not)."""
    print("[case] bkv magnitudes", codec, flush=True)
    bs, hd, heads = 16, 64, 2
    g = np.random.default_rng(5)
    scales = [0.0, 1e-45, 1e-38, 2.0 ** -101, 2.0 ** -100, 1e-20, 1.0, 3e10, 1e38, 3.4e38, np.inf, np.nan, 1.0]
    p = Pair(ctx, 1, heads, hd, 1, bs * len(scales), bs, len(scales), bs * len(scales), codec)
    x = g.uniform(-1, 1, (2, len(scales), bs, heads, hd))
    # values that fall on the middle of two steps under a largest value of 127 or 448
    top = 127 if codec == 0 else 448
    mids = np.concatenate([np.arange(-126, 126) + 0.5, 2.0 ** -10 * np.arange(-40, 41), 17 + 2.0 * np.arange(-9, 9)])
    x[0, 6, :, 0] = 0
    x[0, 6, 0, 0, 0] = top
    x[0, 6].reshape(-1)[hd * heads:hd * heads + mids.size] = mids
    x[0, 6, 1:, 1] = 0
    x[0, 6].reshape(bs, heads, hd)[1:7, 0] = np.resize(mids, (6, hd))
    with np.errstate(invalid="ignore", over="ignore"):
        for i, s in enumerate(scales):
            if np.isfinite(s):
                x[:, i] *= 1.0 if i == 6 else s
            else:
                x[:, i, 3, 1, 9] = s
    k, v = (x[j].reshape(-1, heads * hd).astype(np.float32) for j in (0, 1))
    p.ref.step([0], [0], [len(k)])
    p.dev.step([0], [0], [len(k)])
    p.dev.write(0, k, v)
    p.ref.write(0, k, v)
    p.check_rows()


def test_planning_in_lockstep(ctx):
    """Random steps with take-backs, forks, frees, copies and compactions, valid
    and not: the same outcome, pages, lengths and rows as the restatement."""
    print("[case] bkv lockstep", flush=True)
    a = Pair(ctx, 2, 1, 64, 7, 150, 16, 37, 400, 0, seed=11)
    b = Pair(ctx, 2, 1, 64, 5, 100, 16, 19, 64, 0, seed=12)
    g = np.random.default_rng(3)
    seen = set()
    for i in range(220):
        p = a if g.random() < 0.7 else b
        r, what = p.ref, g.choice(["step", "step", "step", "fork", "free", "copy", "compact"], p=None)
        print("[case] bkv lockstep", i, what, flush=True)
        n = int(g.integers(1, 4))
        ids = g.permutation(np.arange(-1, r.n_seq + 1) if g.random() < 0.15 else np.arange(r.n_seq))[:n]
        if what == "step":
            if g.random() < 0.1:
                ids = np.r_[ids, ids[:1]]
            lens = np.array([r.len[s] if 0 <= s < r.n_seq else 0 for s in ids])
            back = np.where(g.random(ids.size) < 0.4, g.integers(0, 30, ids.size), 0)
            starts = np.maximum(lens - back, 0)
            counts = g.integers(0, 45 if p is a else 12, ids.size)
            if g.random() < 0.1:
                starts[-1] += 1
            if g.random() < 0.05:
                counts[0] = -1
            p.step(ids, starts, counts)
        elif what == "fork":
            dst = g.integers(0, r.n_seq, ids.size) if g.random() < 0.3 else \
                np.resize([s for s in range(r.n_seq) if r.len[s] == 0 and s not in ids] or [0], ids.size)
            p.both("fork", ids, dst)
        elif what == "free":
            p.both("free", np.r_[ids, ids[:1]])
        elif what == "copy":
            q = a if g.random() < 0.5 else b
            src = g.permutation(q.ref.n_seq)[:n]
            dst = np.resize([s for s in range(r.n_seq) if r.len[s] == 0] or [0], src.size)
            want, _ = r.copy_from(q.ref, src, dst)
            assert p.outcome(lambda: p.dev.copy_from(q.dev, src, dst)) == want
        else:
            r.compact()
            p.dev.compact()
        seen.add((what, p.dev is a.dev))
        p.check_state()
        if i % 10 == 9:
            a.check_rows()
            b.check_rows()
    assert len(seen) >= 9


def test_take_back_reaches_the_block_before_and_no_further(ctx):
    print("[case] bkv take back", flush=True)
    bs = 16
    p = Pair(ctx, 1, 2, 64, 3, 200, bs, 20, 200)
    p.step([0], [0], [70])  # blocks 0..3 full, 4 open: rows 48.. may be taken back
    p.step([0], [47], [1])
    p.step([0], [48], [3])
    p.check_state()
    p.check_rows()
    p.both("fork", [0], [1])
    p.step([1], [47], [1])  # a fork goes back to its last full block's end
    p.step([1], [48], [20])
    p.step([0], [50], [20])
    p.check_state()
    p.check_rows()


ATTN = [  # codec, bs, hd, heads, kv heads, lens, counts
    (0, 16, 64, 1, 1, [1], [1]),
    (0, 16, 128, 2, 1, [1, 2, 15, 16, 17, 31, 32, 33], [1] * 8),
    (1, 32, 64, 8, 2, [33, 64, 1, 97], [1, 1, 1, 1]),
    (0, 64, 128, 20, 4, [63, 64, 65, 300], [1, 1, 1, 1]),
    (1, 16, 128, 16, 2, [700, 5], [1, 1]),
    (0, 16, 64, 6, 2, [40, 18, 7], [3, 0, 7]),
    (1, 64, 128, 8, 8, [129, 200], [16, 2]),
    (0, 32, 128, 7, 1, [75, 64], [5, 9]),
    (0, 16, 128, 4, 2, [150, 90, 17], [150, 33, 17]),
    (1, 32, 64, 12, 3, [260, 64], [129, 64]),
    (0, 64, 64, 5, 1, [201], [77]),
    (1, 16, 128, 24, 1, [90], [40]),
    (0, 16, 64, 40, 20, [1100], [1]),
    (0, 16, 128, 32, 1, [50, 900], [1, 1]),
    (0, 16, 128, 4, 1, [9000, 20], [1, 1]),
    (1, 32, 64, 32, 1, [6001], [1]),
    (0, 16, 64, 8, 2, [6500, 300], [16, 9]),
    (1, 64, 128, 32, 1, [7000, 90], [1, 1]),
    (0, 32, 128, 16, 2, [5000], [11]),
    (0, 16, 64, 20, 20, [1000, 300, 31, 640], [900, 0, 31, 600]),
    (1, 32, 128, 16, 1, [5, 2300, 77], [5, 400, 77]),
    (0, 32, 64, 3, 1, [64, 3, 500, 90] * 20, [50, 3, 1, 0] * 20),
]


@pytest.mark.parametrize("codec,bs,hd,heads,kvh,lens,counts", ATTN)
def test_attention(ctx, codec, bs, hd, heads, kvh, lens, counts):
    print("[case] bkv attn", codec, bs, hd, heads, kvh, lens, counts, flush=True)
    n = len(lens)
    p = Pair(ctx, 2, kvh, hd, n, max(lens), bs, sum(lens) // bs + n, sum(lens), codec, seed=sum(lens))
    lens, counts = np.array(lens), np.array(counts)
    p.step(np.arange(n), np.zeros(n, int), lens - counts)
    rows = p.step(np.arange(n), lens - counts, counts)
    for layer in (1, 0):
        got = p.check_attn(layer, rows, heads)
    assert np.all(np.isfinite(got))


@pytest.mark.parametrize("codec,bs,hd,heads,kvh,lens,counts", ATTN + [
    (0, 16, 128, 16, 2, [1500, 700], [1400, 300]), (1, 64, 64, 5, 5, [1, 2, 640], [1, 2, 600]),
    (0, 16, 128, 24, 1, [900, 300, 40, 65], [200, 1, 1, 2])])
@pytest.mark.parametrize("far", [False, True])
def test_attention_of_steps_that_may_be_larger(ctx, codec, bs, hd, heads, kvh, lens, counts, far):
    """The same under bounds far above the step's rows, which lay its work out by
    shares of all workgroups (and, far, items of few rows in a launch of their own);
    rows behind the step's stay as they are."""
    print("[case] bkv attn shares", codec, bs, hd, heads, kvh, lens, counts, far, flush=True)
    n, room = len(lens), 1 << 20
    p = Pair(ctx, 1, kvh, hd, n, 1 << 20 if far else max(max(lens), 64), bs, sum(lens) // bs + n, room, codec, seed=sum(lens))
    lens, counts = np.array(lens), np.array(counts)
    p.step(np.arange(n), np.zeros(n, int), lens - counts)
    assert p.ref.step(list(range(n)), list(lens - counts), list(counts)) == (bm.OK, n)
    p.dev.step_dev(n, room, room, 1 << 24, *(_Ids(ctx, a) for a in (np.arange(n), lens - counts, counts)))
    assert p.dev.status() == n
    rows = int(counts.sum())
    k, v = p.rows(rows)
    q = p.g.standard_normal((rows, heads * hd)).astype(np.float32) * 2
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    out = up(np.full((rows + 1) * heads * hd, 7.5, np.float32))
    p.dev.write_dev(0, up(k), up(v))
    p.ref.write(0, k, v)
    p.dev.attn_dev(0, heads, up(q), hd ** -0.5, out)
    ctx.synchronize()
    got = out.download(np.float32, (rows + 1) * heads * hd).reshape(rows + 1, heads * hd)
    want, tol = p.ref.attn(0, q, heads, np.float32(hd ** -0.5))
    err = np.abs(got[:rows].astype(np.float64) - want) / tol
    assert np.nanmax(err) <= 1 and not np.isnan(err).any()
    assert np.all(got[rows] == 7.5)


def test_attention_of_large_small_and_zero_values(ctx):
    """Scales far apart between blocks and heads, zero blocks, query rows of every
    size: no overflow, and small blocks keep their bits beside large ones."""
    print("[case] bkv attn scales", flush=True)
    bs, hd, kvh, t = 16, 64, 2, 16 * 7 + 5
    for codec in (0, 1):
        p = Pair(ctx, 1, kvh, hd, 1, t, bs, 8, t, codec)
        g = p.g
        p.ref.step([0], [0], [t])
        p.dev.step([0], [0], [t])
        size = np.repeat([1.0, 1e-6, 0.0, 30.0, 1e-30, 1e4, 1.0, 1e-3], bs)[:t, None]
        k = (g.standard_normal((t, kvh * hd)) * np.minimum(size, 30)).astype(np.float32)
        v = (g.standard_normal((t, kvh * hd)) * size).astype(np.float32)
        p.dev.write(0, k, v)
        p.ref.write(0, k, v)
        q = (g.standard_normal((t, 4 * hd)) * np.exp(g.uniform(-60, 0, (t, 1)))).astype(np.float32)
        q[3] = 0
        p.check_attn(0, t, 4, 0.125, q)
        q = g.standard_normal((t, 4 * hd)).astype(np.float32) * 1e30
        p.check_attn(0, t, 4, 1e-30, q)


def test_attention_where_values_are_not_finite(ctx):
    """A NaN or infinity reaches exactly the rows that attend to it: those at and
    after it in the open block, those that see its block once it is full."""
    print("[case] bkv attn nan", flush=True)
    bs, hd, heads = 16, 64, 2
    for at, bad in ((20, np.nan), (20, np.inf), (37, np.nan)):  # 20: a full block's row, 37: the open block's
        t = 40
        p = Pair(ctx, 1, heads, hd, 1, t, bs, 4, t)
        p.ref.step([0], [0], [t])
        p.dev.step([0], [0], [t])
        k, v = p.rows(t)
        v[at, 5] = bad  # head 0
        p.dev.write(0, k, v)
        q = p.g.standard_normal((t, heads * hd)).astype(np.float32)
        got = p.dev.attn(0, q, heads, 0.125).reshape(t, heads, hd)
        assert np.all(np.isfinite(got[:, 1]))
        if at < 32:  # the whole block is NaN
            assert np.all(np.isfinite(got[:16, 0])) and np.all(np.isnan(got[16:, 0]))
        else:
            assert np.all(np.isfinite(got[:at, 0])) and np.all(~np.isfinite(got[at:, 0, 5]))
            assert np.all(np.isfinite(got[:, 0, :5])) and np.all(np.isfinite(got[:, 0, 6:]))
    # a query row that is not finite gives NaN in its own head and row alone
    p = Pair(ctx, 1, heads, hd, 1, 40, bs, 4, 40)
    p.step([0], [0], [40])
    q = p.g.standard_normal((40, heads * hd)).astype(np.float32)
    q[7, 3], q[9, hd + 3] = np.nan, np.inf
    got = p.dev.attn(0, q, heads, 0.125).reshape(40, heads, hd)
    bad = np.zeros((40, heads), bool)
    bad[7, 0] = bad[9, 1] = True
    assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)


def test_the_order_of_a_batch_does_not_matter(ctx):
    """Decode rows of four sequences in two orders: the same bits."""
    print("[case] bkv attn batch", flush=True)
    p = Pair(ctx, 1, 2, 128, 4, 700, 16, 100, 1500)
    lens = np.array([700, 33, 260, 1])
    p.step(np.arange(4), np.zeros(4, int), lens - 1)
    k, v = p.rows(4)
    q = p.g.standard_normal((4, 16 * 128)).astype(np.float32)
    outs = []
    for order in ([0, 1, 2, 3], [3, 1, 0, 2]):
        p.dev.step(order, lens[order] - 1, [1] * 4)
        p.dev.write(0, k[order], v[order])
        out = p.dev.attn(0, q[order], 16, 0.1)
        outs.append(out[np.argsort(order)])
    assert np.array_equal(outs[0], outs[1])


def test_failed_items_leave_their_rows_and_sequences(ctx):
    """A step that ends early: earlier items are done, the rest untouched."""
    print("[case] bkv failed items", flush=True)
    p = Pair(ctx, 1, 1, 64, 4, 64, 16, 5, 128)
    p.step([0, 1, 2, 3], [0, 0, 0, 0], [20, 20, 20, 20])
    n = p.step([0, 1, 2, 3], [20, 20, 20, 20], [12, 11, 44, 1])  # one page is left, item 2 needs three
    p.check_attn(0, n, 2)
    p.check_state()
    p.check_rows()
    n = p.step([0, 0, 1], [32, 32, 31], [1, 1, 1])  # named twice
    p.check_attn(0, n, 1)
    p.both("free", [1])
    q = np.ones((n, 64), np.float32)
    assert np.array_equal(p.dev.attn(0, q, 1, 1.0, out=q * 3), q * 3)  # a free ends the step
    p.check_rows()


def test_beams_over_one_prompt(ctx):
    """Fork, step, attention, free, over several rounds: every beam as if its
    sequence were its own; all pages come back."""
    print("[case] bkv beams", flush=True)
    p = Pair(ctx, 2, 2, 64, 9, 120, 16, 40, 64, 1)
    p.step([0], [0], [55])
    beams = np.array([1, 2, 3, 4])
    p.both("fork", [0] * 4, beams)
    for r in range(12):
        lens = np.array([p.ref.len[s] for s in beams])
        n = p.step(beams, lens, [1] * 4)
        p.check_attn(r % 2, n, 4)
        parents = beams[p.g.integers(0, 4, 4)]
        spare = np.array([s for s in range(1, 9) if s not in beams])[:4]
        p.both("fork", parents, spare)
        p.both("free", beams)
        beams = spare
        p.check_state()
    p.check_rows()
    p.both("free", np.r_[0, beams])
    p.check_state()
    assert p.dev.pages() == (40, 0)


def test_copy_to_a_smaller_cache_and_compaction(ctx):
    print("[case] bkv copy", flush=True)
    a = Pair(ctx, 2, 2, 64, 6, 100, 16, 30, 400, 1)
    a.step(np.arange(6), [0] * 6, [10, 50, 33, 64, 80, 16])
    b = Pair(ctx, 2, 2, 64, 4, 80, 16, 11, 100, 1)
    for src, dst in (([4, 1], [2, 0]), ([2, 0], [1, 1]), ([2], [1]), ([3], [3])):  # named twice; then no pages
        want, _ = b.ref.copy_from(a.ref, src, dst)
        assert b.outcome(lambda: b.dev.copy_from(a.dev, src, dst)) == want
        b.check_state()
    b.both("free", [2])
    b.ref.compact()
    b.dev.compact()
    b.check_state()
    assert max(x for t in b.ref.table for x in t) == b.dev.pages()[1] - 1
    lens = [b.ref.len[0], b.ref.len[1]]
    n = b.step([0, 1], [lens[0] - 3, lens[1]], [4, 2])  # copies can be taken back like their source
    b.check_attn(1, n, 2)
    b.check_rows()
    a.check_rows()


def test_a_step_is_written_where_compaction_has_moved_its_pages(ctx):
    print("[case] bkv compact in a step", flush=True)
    p = Pair(ctx, 2, 2, 64, 3, 200, 16, 20, 200)
    p.step([0, 1], [0, 0], [160, 20])
    p.both("free", [0])
    p.step([1, 2], [20, 0], [0, 100])
    p.both("free", [1])
    p.step([0, 2], [0, 100], [40, 30], write=False)
    p.ref.compact()
    p.dev.compact()
    for layer in range(2):
        k, v = p.rows(70)
        p.dev.write(layer, k, v)
        p.ref.write(layer, k, v)
        p.check_attn(layer, 70, 2)
    p.check_state()
    p.check_rows()


@pytest.mark.parametrize("count,kvh", [(1, 2), (2, 1), (9, 1)])
def test_captured_calls_pass_over_a_larger_step(ctx, count, kvh):
    """write and attn of a graph meet steps of more items, rows, or rows an item
    than the step before the capture: they do what fits and nothing else."""
    print("[case] bkv graph small", count, kvh, flush=True)
    heads, hd, n = 8, 64, 3
    p = Pair(ctx, 1, kvh, hd, 6, 300, 16, 100, 450)
    p.step(np.arange(6), np.zeros(6, int), [100, 37, 64, 5, 150, 80])
    lens = np.array(p.ref.len)
    rows, w, wq = n * count, kvh * hd, heads * hd
    p.step(np.arange(n), lens[:n], [count] * n)
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    xs = [p.g.standard_normal((rows, x)).astype(np.float32) for x in (w, w, wq)]
    k, v, q = (up(x) for x in xs)
    mark = np.full((rows + 4) * wq, 7.5, np.float32)
    o = up(mark)

    def body():
        p.dev.write_dev(0, k, v)
        p.dev.attn_dev(0, heads, q, 0.125, o)

    body()
    p.ref.write(0, xs[0], xs[1])
    graph = ctx.capture(body)
    for counts in ([count] * 6, [count, count + 1, count - 1], [5 * count, 1, 1], [count] * n):
        m = len(counts)
        p.step(np.arange(m), p.ref.len[:m], counts, write=False)
        o.upload(mark)
        graph.launch()
        ctx.synchronize()
        got = o.download(np.float32, mark.size)
        assert np.all(got[rows * wq:] == 7.5)
        if counts == [count] * n:
            p.ref.write(0, xs[0], xs[1])
            want, tol = p.ref.attn(0, xs[2], heads, np.float32(0.125))
            assert np.all(np.abs(got[:rows * wq].reshape(rows, wq) - want) <= tol)
        kk, vv = p.rows(sum(counts))
        p.dev.write(0, kk, vv)
        p.ref.write(0, kk, vv)
        p.check_attn(0, sum(counts), heads)
    p.check_rows()


def test_more_pages_than_32_bits_of_bytes(ctx):
    """A pool of over 4 GiB: the last pages hold what the first ones do."""
    print("[case] bkv large pool", flush=True)
    bs, hd, heads, n_page = 64, 128, 8, 36000  # 131 KB a page
    kv = ctx.block_kv_cache(1, heads, hd, 3, 1 << 22, bs, n_page, 1 << 20)
    g = np.random.default_rng(0)
    # sequence 0 fills the pool but for a few pages without any data of its own
    at = 0
    while at < (n_page - 4) * bs:
        n = min(1 << 20, (n_page - 4) * bs - at)
        kv.step([0], [at], [n])
        at += n
    assert kv.pages() == (4, n_page - 4)
    x = [g.standard_normal((200, heads * hd)).astype(np.float32) for _ in (0, 1)]
    q = g.standard_normal((200, heads * hd)).astype(np.float32)
    kv.step([1], [0], [200])
    assert kv.page_of(1, 2) == n_page - 2
    kv.write(0, *x)
    out = kv.attn(0, q, heads, 0.1)
    rows = kv.read(0, np.full(200, 1), np.arange(200))
    kv.free([0])
    kv.step([2], [0], [200])
    assert kv.page_of(2, 2) == 2
    kv.write(0, *x)
    assert np.array_equal(kv.attn(0, q, heads, 0.1), out)
    low = kv.read(0, np.full(200, 2), np.arange(200))
    assert np.array_equal(low[0], rows[0]) and np.array_equal(low[1], rows[1])
    kv.compact()
    assert kv.page_of(1, 2) < 6
    again = kv.read(0, np.full(200, 1), np.arange(200))
    assert np.array_equal(again[0], rows[0]) and np.array_equal(again[1], rows[1])


def test_a_captured_step_replays_with_what_the_arrays_hold(ctx):
    """free, fork, step, write and attn in one graph, replayed as the device
    arrays change, with eager calls between: equal to the eager calls."""
    print("[case] bkv graph", flush=True)
    heads, hd, kvh = 4, 64, 2
    w, wq = kvh * hd, heads * hd
    p = Pair(ctx, 2, kvh, hd, 6, 400, 16, 120, 300)
    p.step([0, 1], [0, 0], [90, 200])
    src, dst = _Ids(ctx, [0, 1, 1, 0]), _Ids(ctx, [2, 3, 4, 5])
    starts, counts = _Ids(ctx, [90, 200, 200, 90]), _Ids(ctx, [2, 1, 0, 1])
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    k, v = (up(np.zeros((4, w), np.float32)) for _ in (0, 1))
    q, o = up(np.zeros((4, wq), np.float32)), up(np.zeros((4, wq), np.float32))

    def body():
        p.dev.free_dev(4, dst)
        p.dev.fork_dev(4, src, dst)
        p.dev.step_dev(4, 4, 2, 260, dst, starts, counts)
        for layer in (0, 1):
            p.dev.write_dev(layer, k, v)
        p.dev.attn_dev(1, heads, q, 0.125, o)

    body()
    graph = ctx.capture(body)
    g = np.random.default_rng(2)
    for i in range(5):
        s = g.integers(0, 2, 4)
        lens = np.array([p.ref.len[x] for x in s])
        cnt = np.array([[2, 1, 0, 1], [1, 1, 1, 1], [0, 2, 2, 0]][i % 3])
        src.b.upload(s.astype(np.int32))
        starts.b.upload(lens.astype(np.int32))
        counts.b.upload(cnt.astype(np.int32))
        xs = [g.standard_normal((4, n)).astype(np.float32) for n in (w, w, wq)]
        for buf, x in zip((k, v, q), xs):
            buf.upload(x)
        graph.launch()
        ctx.synchronize()
        assert p.dev.status() == 4
        p.ref.free([2, 3, 4, 5])
        p.ref.fork(list(s), [2, 3, 4, 5])
        p.ref.step([2, 3, 4, 5], list(lens), list(cnt))
        for layer in (0, 1):
            p.ref.write(layer, xs[0], xs[1])
        want, tol = p.ref.attn(1, xs[2], heads, np.float32(0.125))
        got = o.download(np.float32, 4 * wq).reshape(4, wq)
        n = int(cnt.sum())
        assert np.all(np.abs(got[:n] - want[:n]) <= tol[:n])
        p.check_state()
        if i == 2:  # eager work between replays
            p.step([0], [p.ref.len[0]], [5])
    p.check_rows()


def test_refusals(ctx):
    print("[case] bkv refusals", flush=True)
    ok = (1, 2, 64, 3, 100, 16, 10, 64)
    for i in range(8):
        bad = list(ok)
        bad[i] = 0
        with pytest.raises(hip.InvalidArgument):
            ctx.block_kv_cache(*bad)
    for i, x in ((2, 96), (5, 17), (5, 128)):
        bad = list(ok)
        bad[i] = x
        with pytest.raises(hip.UnsupportedOp):
            ctx.block_kv_cache(*bad)
    with pytest.raises(hip.UnsupportedOp):
        ctx.block_kv_cache(*ok, codec=7)
    for i, x in ((0, 5000), (1, 2000), (3, 70000), (4, 1 << 25), (6, 1 << 27), (7, 1 << 21)):
        bad = list(ok)
        bad[i] = x
        with pytest.raises(hip.InvalidArgument):
            ctx.block_kv_cache(*bad)
    kv = ctx.block_kv_cache(*ok)
    other = ctx.block_kv_cache(1, 2, 64, 3, 100, 32, 10, 64)
    with pytest.raises(hip.InvalidArgument):
        kv.copy_from(other, [0], [0])
    with pytest.raises(hip.InvalidArgument):
        kv.step([0], [0], [65])  # over max_rows: refused as a whole
    assert kv.length(0) == 0
    with pytest.raises(hip.InvalidArgument):
        kv.step(np.arange(1025), np.zeros(1025), np.zeros(1025))
    kv.step([0], [0], [5])
    x = np.ones((5, 128), np.float32)
    for call in (lambda: kv.write(1, x, x), lambda: kv.attn(1, x, 2, 1.0), lambda: kv.read(1, [0], [0]),
                 lambda: kv.attn(0, np.ones((5, 192), np.float32), 3, 1.0), lambda: kv.write(0, x[:4], x),
                 lambda: kv.length(3), lambda: kv.step([0, 1], [0], [1])):
        with pytest.raises(hip.InvalidArgument):
            call()
    b = hip.DeviceBuffer.from_array(ctx, np.zeros(4096, np.float32))
    off = type("P", (), {"ptr": hip.C.c_void_p(b.ptr.value + 4)})()
    null = type("P", (), {"ptr": hip.C.c_void_p()})()
    for bad in (off, null):
        for call in (lambda: kv.write_dev(0, bad, b), lambda: kv.write_dev(0, b, bad),
                     lambda: kv.attn_dev(0, 2, bad, 1.0, b), lambda: kv.attn_dev(0, 2, b, 1.0, bad),
                     lambda: kv.read_dev(0, 1, b, b, bad, b), lambda: kv.read_dev(0, 1, b, b, b, bad)):
            with pytest.raises(hip.InvalidArgument):
                call()
    for call in (lambda: kv.step_dev(1, 1, 1, 1, null, b, b), lambda: kv.fork_dev(1, null, b),
                 lambda: kv.free_dev(1, null), lambda: kv.copy_from_dev(kv, 1, b, null),
                 lambda: kv.step_dev(1, 65, 1, 1, b, b, b), lambda: kv.free_dev(1025, b)):
        with pytest.raises(hip.InvalidArgument):
            call()
    kv.reset()
    assert kv.pages() == (10, 0) and kv.length(0) == 0
    assert np.array_equal(kv.attn(0, x, 2, 1.0, out=x * 2), x * 2)  # nothing is planned
    kv.step([], [], [])
    kv.write(0, x[:0], x[:0])
