"""Reordering of the paged Q8_0 cache's streams, and of the sessions that hold one: rows are moved, not
computed, so everything is compared bit for bit with what the streams held before."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_sessions import make_decoder
from tests.test_gpu_textdec import build
from vokra_amd import hip

F = np.float32


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def filled(ctx, g, layers, h, hd, streams, max_time, bs, lens):
    """A cache whose stream s holds lens[s] rows of each layer, on shuffled pages."""
    kv = hip.KvCache(ctx, layers, h, hd, streams, max_time, bs)
    free, _ = kv.pages()
    kv.set_free_order(g.permutation(free))
    for layer in range(layers):
        st = np.concatenate([np.full(n, s) for s, n in enumerate(lens)] + [[]]).astype(np.int32)
        tt = np.concatenate([np.arange(n) for n in lens] + [[]]).astype(np.int32)
        for a in range(0, st.size, 1024):
            i = slice(a, a + 1024)
            rows = [(g.standard_normal((st[i].size, h * hd)) * 2).astype(F) for _ in (0, 1)]
            kv.append(layer, st[i], tt[i], *rows)
    return kv


def held(kv, layers, streams, max_time):
    """[layer, stream, side, time, width]; NaN where there is no page."""
    out = np.full((layers, streams, 2, max_time, kv.width), np.nan, F)
    for layer in range(layers):
        for s in range(streams):
            for t in range(max_time):
                r = kv.read(layer, t, s)
                if r is not None:
                    out[layer, s, :, t] = r
    return out


def reordered(before, streams, parents, lens):
    after = before.copy()
    for g, n in enumerate(lens):
        for s, p in zip(streams[g], parents[g]):
            if p >= 0:
                after[:, s, :, :n] = before[:, streams[g][p], :, :n]
    return after


@pytest.mark.gpu
@pytest.mark.parametrize("h,hd,bs,layers,groups,beams,max_time", [
    (2, 64, 16, 2, 2, 5, 37), (1, 128, 32, 1, 1, 2, 64), (3, 64, 5, 1, 3, 4, 23), (1, 64, 1, 2, 1, 3, 7),
    (2, 128, 16, 1, 2, 8, 33), (1, 64, 16, 1, 1, 9, 17), (1, 64, 7, 1, 2, 16, 15), (1, 128, 4, 1, 1, 17, 9),
    (1, 64, 16, 1, 1, 32, 18), (20, 64, 16, 1, 1, 5, 20)])
def test_rows_move_as_they_were(ctx, h, hd, bs, layers, groups, beams, max_time):
    print("[case] reorder", h, hd, bs, layers, groups, beams, max_time, flush=True)
    g = np.random.default_rng(beams)
    n = groups * beams + 2  # two streams that no group names
    kv = filled(ctx, g, layers, h, hd, n, max_time, bs, np.full(n, max_time))
    ids = g.permutation(n)[:groups * beams].reshape(groups, beams)
    before = held(kv, layers, n, max_time)
    kinds = [np.tile(np.arange(beams), (groups, 1)),  # everyone stays
             np.tile(np.roll(np.arange(beams), 1), (groups, 1)),  # one cycle
             np.tile(np.arange(beams)[::-1], (groups, 1)),  # swaps
             np.full((groups, beams), beams - 1),  # all from one
             g.integers(-1, beams, (groups, beams)), g.integers(-1, beams, (groups, beams))]
    for parents in kinds:
        lens = g.integers(0, max_time + 1, groups)
        lens[0] = g.choice([max_time, max_time // bs * bs, min(bs, max_time), 1])
        pages = kv.pages()
        kv.reorder(ids, parents, lens)
        after = held(kv, layers, n, max_time)
        assert np.array_equal(after, reordered(before, ids, parents, lens))
        assert kv.pages() == pages
        before = after


@pytest.mark.gpu
def test_lengths_of_none_and_pages_that_are_not_there(ctx):
    print("[case] reorder lengths", flush=True)
    g = np.random.default_rng(0)
    kv = filled(ctx, g, 2, 1, 64, 4, 40, 16, [9, 9, 9, 9])
    before = held(kv, 2, 4, 40)
    kv.reorder([[0, 1, 2, 3]], [[1, 0, 0, 2]], [0])
    assert np.array_equal(held(kv, 2, 4, 40), before, equal_nan=True)
    kv.reorder([[0, 1, 2, 3]], [[1, 0, 0, 2]], [40])  # longer than what is held: only pages there are move
    want = reordered(before, [[0, 1, 2, 3]], [[1, 0, 0, 2]], [16])
    assert np.array_equal(held(kv, 2, 4, 40), want, equal_nan=True)
    kv.reorder(np.zeros((0, 4), np.int32), np.zeros((0, 4), np.int32), [])


def _up(ctx, a):
    return hip.DeviceBuffer.from_array(ctx, np.asarray(a, np.int32))


@pytest.mark.gpu
def test_device_items_that_name_nothing_are_passed_over_and_graphs(ctx):
    print("[case] reorder device", flush=True)
    g = np.random.default_rng(1)
    n, t = 9, 21
    kv = filled(ctx, g, 2, 2, 64, n, t, 8, np.full(n, t))
    before = held(kv, 2, n, t)
    ids = np.array([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    d_ids, d_par, d_len = _up(ctx, ids), _up(ctx, np.zeros((3, 3))), _up(ctx, [0, 0, 0])

    def put(ids, par, lens):
        for b, a in ((d_ids, ids), (d_par, par), (d_len, lens)):
            b.upload(np.asarray(a, np.int32))
    # group 0: parents out of range; group 1: longer than max_len, group 2: a stream out of range on either side
    put([[0, 1, 2], [3, 4, 5], [6, 9, -1]], [[2 ** 31 - 1, -2 ** 31, 3], [1, 2, 0], [1, 0, 0]], [t, t, t])
    kv.reorder_dev(3, 3, d_ids, d_par, d_len, t - 1)
    ctx.synchronize()
    assert np.array_equal(held(kv, 2, n, t), before)
    kv.reorder_dev(3, 3, d_ids, d_par, d_len, t)
    ctx.synchronize()
    want = reordered(before, [[3, 4, 5]], [[1, 2, 0]], [t])
    assert np.array_equal(held(kv, 2, n, t), want)
    put(ids, [[1, 2, 0], [1, 0, 0], [0, 1, 2]], [-5, 2 ** 31 - 1, 7])
    kv.reorder_dev(3, 3, d_ids, d_par, d_len, t)
    ctx.synchronize()
    assert np.array_equal(held(kv, 2, n, t), want)
    put(ids, [[1, 2, 0], [1, 0, 0], [2, 0, 1]], [-2 ** 31, -2 ** 31 + 8, -1])  # below zero by as much as there is
    kv.reorder_dev(3, 3, d_ids, d_par, d_len, t)
    ctx.synchronize()
    assert np.array_equal(held(kv, 2, n, t), want)
    graph = ctx.capture(lambda: kv.reorder_dev(3, 3, d_ids, d_par, d_len, t))
    for _ in range(3):
        par, lens = g.integers(-1, 3, (3, 3)), g.integers(0, t + 1, 3)
        put(ids, par, lens)
        graph.launch()
        ctx.synchronize()
        want = reordered(want, ids, par, lens)
        assert np.array_equal(held(kv, 2, n, t), want)


@pytest.mark.gpu
def test_decoder_beams_go_on_from_their_parents(ctx, oracle):
    """A stream's step after a reorder is the step of a stream that read the same tokens itself, bit for bit."""
    print("[case] decoder reorder", flush=True)
    a, _ = make_decoder(ctx, oracle, np.random.default_rng(5))
    b, _ = make_decoder(ctx, oracle, np.random.default_rng(5))
    for dec in (a, b):
        for s in range(4):  # beams of one utterance
            dec.set_encoder(s, a.parts["encs"][0])
    g = np.random.default_rng(6)
    a.step([2], [7], [0])
    with pytest.raises(hip.InvalidArgument):  # the other streams have read nothing
        a.step([0], [9], [1])
    a.reorder([[2, 0, 3, 1]], [[0, 0, 0, 0]])
    read = [[7] for _ in range(4)]
    for step in range(1, 9):
        tok = g.integers(0, 300, 4)
        _, la = a.step([0, 1, 2, 3], tok, [step] * 4, want_logits=True)
        for s in range(4):
            read[s].append(int(tok[s]))
        b.reset()
        for t in range(step + 1):
            _, lb = b.step([0, 1, 2, 3], [r[t] for r in read], [t] * 4, want_logits=True)
        assert np.array_equal(la, lb), step
        parents = g.integers(-1, 4, (1, 4))
        ids = g.permutation(4)[None]
        a.reorder(ids, parents)
        old = [list(r) for r in read]
        for s, p in zip(ids[0], parents[0]):
            read[s] = list(old[ids[0, p]] if p >= 0 else old[s])
    with pytest.raises(hip.InvalidArgument):
        a.reorder([[0, 0]], [[0, 1]])


@pytest.mark.gpu
def test_text_decoder_beams_go_on_from_their_parents(ctx, oracle):
    print("[case] text decoder reorder", flush=True)
    mk = lambda: build(ctx, oracle, 3, 2, 256, 4, 2, 64, 512, 96, 64, 4, bs=4)[0]  # noqa: E731
    a, b = mk(), mk()
    g = np.random.default_rng(8)
    read = [[] for _ in range(4)]
    for step in range(7):
        tok = g.integers(0, 96, 4)
        for s in range(4):
            read[s].append(int(tok[s]))
        _, la = a.step([0, 1, 2, 3], tok, want_logits=True)
        b.reset()
        for t in range(step + 1):
            _, lb = b.step([0, 1, 2, 3], [r[t] for r in read], want_logits=True)
        assert np.array_equal(la, lb), step
        parents = g.integers(0, 2, (2, 2))
        a.reorder([[0, 3], [2, 1]], parents)
        old = [list(r) for r in read]
        for ids, par in zip(([0, 3], [2, 1]), parents):
            for s, p in zip(ids, par):
                read[s] = list(old[ids[p]])
    # streams at different positions: a beam takes its parent's
    a.step([0, 1], [1, 2])
    a.reorder([[0, 2]], [[1, 1]])
    assert [a.position(s) for s in range(4)] == [7, 8, 7, 7]
    # through the device forms, the lengths the caller's
    d = [_up(ctx, x) for x in ([[3, 1]], [[1, 0]], [8])]
    a.reorder_dev(1, 2, *d, 8)
    ctx.synchronize()


@pytest.mark.gpu
def test_refusals(ctx):
    print("[case] reorder refusals", flush=True)
    kv = hip.KvCache(ctx, 1, 1, 64, 6, 32, 16)

    def bad(*a):
        with pytest.raises(hip.InvalidArgument):
            kv.reorder(*a)
    bad([[0, 1]], [[0, 2]], [1])
    bad([[0, 1]], [[0, -2]], [1])
    bad([[0, 0]], [[0, 1]], [1])
    bad([[0, 6]], [[0, 1]], [1])
    bad([[-1, 2]], [[0, 1]], [1])
    bad([[0, 1]], [[0, 1]], [33])
    bad([[0, 1]], [[0, 1]], [-1])
    bad([[0, 1], [1, 2]], [[0, 1], [0, 1]], [1, 1])
    bad([[0, 1]], [[0, 1]], [1, 1])
    bad([0, 1], [0, 1], [1, 1])
    bad(np.zeros((1, 0)), np.zeros((1, 0)), [1])
    d = _up(ctx, np.zeros(64))
    for args in ((1, 0, d, d, d, 4), (1, 33, d, d, d, 4), (4, 2, d, d, d, 4), (1, 2, d, d, d, 33)):
        with pytest.raises(hip.InvalidArgument):
            kv.reorder_dev(*args)
    big = hip.KvCache(ctx, 1, 1, 64, 40, 32, 16)
    with pytest.raises(hip.InvalidArgument):  # 33 beams
        big.reorder_dev(1, 33, d, d, d, 4)
    ctx.synchronize()


def test_missing_arguments_are_refused_without_a_device():
    L, null = hip.lib(), C.c_void_p()
    for name in ("kv", "decoder", "text_decoder"):
        assert getattr(L, f"vokra_hip_{name}_reorder_dev")(null, null, 1, 1, null, null, null, 1) == 5
    assert L.vokra_hip_kv_reorder(null, null, 1, 1, None, None, None) == 5
    assert L.vokra_hip_decoder_reorder(null, null, 1, 1, None, None) == 5
    assert L.vokra_hip_text_decoder_reorder(null, null, 1, 1, None, None) == 5
