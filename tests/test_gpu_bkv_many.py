"""The block-scaled cache with as many items as a call takes, against bkv_model."""
import numpy as np
import pytest

from tests import bkv_model as bm
from tests.test_gpu_bkv import Pair, _Ids
from vokra_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def test_more_fork_items_than_sequences(ctx):
    """1024 items that name one destination, over many layers and heads: the first is
    forked with its rows, the second is refused."""
    print("[case] bkv fork items", flush=True)
    layers, heads, hd = 64, 512, 64
    kv = ctx.block_kv_cache(layers, heads, hd, 2, 16, 16, 1, 4)
    kv.step([0], [0], [3])
    k = np.random.default_rng(0).standard_normal((2, 3, heads * hd)).astype(np.float32)
    for layer in (0, layers - 1):
        kv.write(layer, *k)
    with pytest.raises(hip.InvalidArgument):
        kv.fork([0] * 1024, [1] * 1024)
    assert kv.length(1) == 3
    for layer in (0, layers - 1):
        for got, want in zip(kv.read(layer, [1] * 3, [0, 1, 2]), k):
            assert np.array_equal(got, want)


@pytest.mark.parametrize("n", [257, 1024])
def test_steps_forks_and_frees_of_many_sequences(ctx, n):
    """Planning by 1024 threads over real items: ragged steps, take-backs, items that
    fail past the 256th, forks of many, frees that name some twice, and attention."""
    print("[case] bkv many", n, flush=True)
    bs, t = 16, 64
    p = Pair(ctx, 1, 1, 64, 2 * n, t, bs, 5 * n, 40 * n, seed=n)
    g = p.g
    ids = g.permutation(2 * n)[:n]
    p.step(ids, np.zeros(n, int), g.integers(0, 41, n))
    p.check_state()
    p.check_rows()
    # take-backs of some, one token for others; attention of all
    lens, floors = (np.array([x[s] for s in ids]) for x in (p.ref.len, p.ref.floor))
    starts = np.where(g.random(n) < 0.4, g.integers(floors, lens + 1), lens)
    counts = np.minimum(g.integers(0, 4, n), t - starts)
    p.step(ids, starts, counts)
    p.check_attn(0, int(counts.sum()), 2)
    # an item past the 256th fails: named twice, too far, an unknown sequence
    for at, (seq, start) in ((256, (ids[3], None)), (n - 1, (ids[n - 1], t + 1)), (n - 2, (2 * n, 0))):
        seqs = ids.copy()
        starts = np.array([p.ref.len[s] for s in seqs])
        counts = np.where(starts < t, 1, 0)
        seqs[at] = seq
        starts[at] = p.ref.len[seq] if start is None else start
        p.step(seqs, starts, counts)
        p.check_attn(0, int(counts.sum()), 2)
    p.check_state()
    # forks into the other half, the last of them into a sequence that is not empty
    rest = np.setdiff1d(np.arange(2 * n), ids)
    p.both("fork", list(ids), list(rest[:n - 1]) + [ids[0]])
    p.check_state()
    p.both("free", list(ids[:n - 9]) + list(ids[:9]))
    p.check_state()
    lens = np.array([p.ref.len[s] for s in rest])
    p.step(rest, lens, np.where(lens < t, 1, 0))
    p.check_attn(0, int((lens < t).sum()), 2)
    p.check_rows()
    p.both("compact")
    p.check_state()
    p.check_rows()


def test_a_step_of_many_items_runs_out_of_pages_past_the_256th(ctx):
    print("[case] bkv many exhausted", flush=True)
    n = 600
    p = Pair(ctx, 1, 1, 64, n, 64, 16, 700, 40 * n)
    p.step(np.arange(n), np.zeros(n, int), p.g.integers(17, 41, n))  # one or two pages an item
    assert 256 < len(p.ref.plan) < n
    p.check_state()
    p.check_rows()


@pytest.mark.parametrize("long_items", [6, 700])
def test_attention_of_many_items_in_shares(ctx, long_items):
    """1000 items, some of them chunks: tiles of 128 columns placed among as many items as a
    call takes, with the single tokens in a launch of their own where they are most."""
    print("[case] bkv many shares", long_items, flush=True)
    n, kvh, heads, hd, top = 1000, 2, 8, 64, 40
    p = Pair(ctx, 1, kvh, hd, n, 400, 16, 4000, n * 64, seed=long_items)
    g = p.g
    lens = g.integers(0, 30, n)
    lens[:2] = 350, 200
    p.step(np.arange(n), np.zeros(n, int), lens)
    counts = np.ones(n, int)
    counts[g.permutation(n)[:long_items]] = g.integers(2, top + 1, long_items)
    counts[0] = top
    p.step(np.arange(n), lens, counts)
    p.check_attn(0, int(counts.sum()), heads)


def test_captured_copies_and_compaction_replay(ctx):
    """copy, compact, read and free in one graph, replayed as the source changes, with
    eager calls on both caches between: equal to the restatement each time."""
    print("[case] bkv graph copy", flush=True)
    args = (2, 2, 64, 5, 200, 16)
    a, b = Pair(ctx, *args, 60, 400), Pair(ctx, *args, 40, 400, seed=1)
    a.step([0, 1, 2], [0, 0, 0], [70, 16, 5])
    b.step([4], [0], [50])
    w, most = 128, 256
    src, dst = _Ids(ctx, [0, 1]), _Ids(ctx, [1, 3])
    seqs, times = _Ids(ctx, np.zeros(most)), _Ids(ctx, np.zeros(most))
    k, v = (hip.DeviceBuffer.from_array(ctx, np.zeros(most * w, np.float32)) for _ in (0, 1))

    def body():
        b.dev.free_dev(2, dst)
        b.dev.compact()
        b.dev.copy_from_dev(a.dev, 2, src, dst)
        b.dev.read_dev(1, most, seqs, times, k, v)

    body()
    graph = ctx.capture(body)
    for i in range(5):
        pair = [(0, 1), (2, 0), (1, 2), (0, 2), (1, 0)][i]
        src.b.upload(np.array(pair, np.int32))
        ids = np.full((2, most), -1, np.int32)
        at = 0
        for s, d in zip(pair, (1, 3)):
            m = a.ref.len[s]
            ids[0, at:at + m] = d
            ids[1, at:at + m] = np.arange(m)
            at += m
        seqs.b.upload(ids[0])
        times.b.upload(ids[1])
        graph.launch()
        ctx.synchronize()
        assert b.dev.status() == 2
        b.ref.free([1, 3])
        b.ref.compact()
        assert b.ref.copy_from(a.ref, list(pair), [1, 3]) == (bm.OK, 2)
        b.check_state()
        held = [b.ref.held(1, d) for d in (1, 3)]
        for side, buf in ((0, k), (1, v)):
            want = np.concatenate([h[side].reshape(-1, w) for h in held] + [np.zeros((most - at, w), np.float32)])
            assert np.array_equal(buf.download(np.float32, most * w).reshape(most, w), want)
        # eager work: the source goes on, the destination's sequences too
        a.step([0, 2], [a.ref.len[0], a.ref.len[2]], [1, 9])
        b.step([1, 4], [b.ref.len[1], b.ref.len[4]], [3, 2])
        b.check_attn(0, 5, 4)
    b.check_rows()
