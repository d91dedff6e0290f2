"""The operators of a generation with several candidates together, as a decoder
calls them: positions by a rotary plan, a step of the block cache with its rows
and attention, the logits rules, and candidates that are forked, taken back,
freed and copied to another cache. Every operator is compared on what it was
given, while its output is what the next one gets."""
import numpy as np
import pytest

from tests import bkv_model as bm
from tests.test_gpu_logits_rules import rules
from tests.test_gpu_rope_plan import check, thetas
from vokra_amd import hip

pytestmark = pytest.mark.gpu
F = np.float32
LAYERS, HQ, KVH, HD, D, VOCAB, ROWS = 2, 6, 2, 64, 96, 997, 64
SCALE = HD ** -0.5


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


class Model:
    """Two layers of attention with random weights; everything between the
    operators is the framework's as well."""

    def __init__(self, ctx, layout, scaling):
        self.ctx, g = ctx, np.random.default_rng(11)
        self.up = lambda a: hip.DeviceBuffer.from_array(ctx, a)

        def weight(k, n):
            return self.up((g.standard_normal((k, n)) / np.sqrt(k)).astype(F))
        self.emb = g.standard_normal((VOCAB, D)).astype(F)
        self.wqk = [weight(D, (HQ + KVH) * HD) for _ in range(LAYERS)]
        self.wv = [weight(D, KVH * HD) for _ in range(LAYERS)]
        self.wo = [weight(HQ * HD, D) for _ in range(LAYERS)]
        self.head, self.gamma = weight(D, VOCAB), self.up(np.ones(D, F))
        self.layout, self.th = layout, thetas(HD, 10000.0, **scaling)
        self.plan = ctx.rope_plan(HD, HD, layout, 10000.0, scaling.get("scaling", hip.RopeScaling.NONE),
                                  scaling.get("factor", 1.0), scaling.get("orig", 0))

        def zeros(*shape):
            return self.up(np.zeros(shape, F))
        self.x, self.h, self.y = zeros(ROWS, D), zeros(ROWS, D), zeros(ROWS, D)
        self.qk, self.q, self.o = ([zeros(ROWS, n * HD) for _ in range(LAYERS)] for n in (HQ + KVH, HQ, HQ))
        self.k, self.v = ([zeros(ROWS, KVH * HD) for _ in range(LAYERS)] for _ in (0, 1))
        self.logits, self.after = zeros(ROWS, VOCAB), zeros(ROWS, VOCAB)
        self.pos, self.seqs, self.starts, self.counts, self.next = (self.up(np.zeros(ROWS, np.int32)) for _ in range(5))

    def bind(self, mask, most):
        """The rules of the next rows, in buffers that stay: up to `most` history ids a call."""
        self.rep, self.freq = self.up(np.full(ROWS, 1.3, F)), self.up(np.full(ROWS, 0.1, F))
        self.hist, self.off = self.up(np.zeros(most, np.int32)), self.up(np.zeros(ROWS + 1, np.int32))
        bits = np.zeros(-(-VOCAB // 32) * 32, np.uint8)
        bits[:VOCAB] = mask
        self.mask = self.up(np.packbits(bits, bitorder="little").view(np.uint32))
        self.rules = hip.LogitsRules(n_hist=most, hist=self.hist, hist_offsets=self.off, repetition=self.rep,
                                     frequency=self.freq, mask=self.mask)

    def put(self, tokens, seqs, starts, counts, history):
        self.x.upload(self.emb[np.asarray(tokens)])
        self.pos.upload(np.concatenate([a + np.arange(n) for a, n in zip(starts, counts)]).astype(np.int32))
        for b, a in ((self.seqs, seqs), (self.starts, starts), (self.counts, counts)):
            b.upload(np.asarray(a, np.int32))
        self.off.upload(np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32))
        self.hist.upload(np.concatenate(history).astype(np.int32))

    def forward(self, cache, n, rows, most, max_len):
        """One call of the model over `rows` packed rows of n sequences; no host work in it."""
        c = self.ctx
        cache.step_dev(n, rows, most, max_len, self.seqs, self.starts, self.counts)
        for i in range(LAYERS):
            c.rms_norm_f32_dev(self.x, self.h, rows, D, self.gamma, 1e-5)
            c.gemm_f32_dev(rows, (HQ + KVH) * HD, D, self.h, self.wqk[i], self.qk[i])
            c.gemm_f32_dev(rows, KVH * HD, D, self.h, self.wv[i], self.v[i])
            k_in = type("At", (), {"ptr": self.qk[i].ptr.value + 4 * HQ * HD})
            w = (HQ + KVH) * HD
            self.plan.apply_dev(rows, self.pos, HQ, self.qk[i], self.q[i], KVH, k_in, self.k[i], q_stride=w, k_stride=w)
            cache.write_dev(i, self.k[i], self.v[i])
            cache.attn_dev(i, HQ, self.q[i], SCALE, self.o[i])
            c.gemm_f32_dev(rows, D, HQ * HD, self.o[i], self.wo[i], self.y)
            c.add_f32_dev(self.x, self.y, self.x, rows * D)
        c.gemm_f32_dev(rows, VOCAB, D, self.x, self.head, self.logits)
        c.logits_rules_dev(rows, VOCAB, self.logits, self.rules, self.after, self.next)

    def got(self, buf, rows, width):
        return buf.download(F, rows * width).reshape(rows, width)

    def outputs(self, rows):
        return [self.got(b, rows, HQ * HD) for b in self.o] + [self.got(self.after, rows, VOCAB),
                                                               self.next.download(np.int32, rows)]

    def compare(self, ref, rows, starts, counts, history, mask):
        """Every operator of the last forward against its definition, on its own inputs."""
        pos = np.concatenate([a + np.arange(n) for a, n in zip(starts, counts)])
        for i in range(LAYERS):
            qk, q, k = (self.got(b[i], rows, n * HD) for b, n in ((self.qk, HQ + KVH), (self.q, HQ), (self.k, KVH)))
            check(q, qk[:, :HQ * HD].reshape(rows, HQ, HD), pos, self.th, self.layout)
            check(k, qk[:, HQ * HD:].reshape(rows, KVH, HD), pos, self.th, self.layout)
            ref.write(i, k, self.got(self.v[i], rows, KVH * HD))
            want, tol = ref.attn(i, q, HQ, F(SCALE))
            err = np.abs(self.got(self.o[i], rows, HQ * HD) - want) / tol
            assert err.max() <= 1, (i, err.max())
        want = rules(self.got(self.logits, rows, VOCAB), history, np.full(rows, 1.3), frequency=np.full(rows, 0.1),
                     mask=mask)
        assert np.array_equal(self.got(self.after, rows, VOCAB), want[0])
        assert np.array_equal(self.next.download(np.int32, rows), want[1])


@pytest.mark.parametrize("codec,layout,scaling", [
    (hip.KvCodec.INT8, hip.RopeLayout.HALF, {}),
    (hip.KvCodec.E4M3, hip.RopeLayout.INTERLEAVED, dict(scaling=hip.RopeScaling.BANDS, factor=8.0, orig=32))])
def test_candidates_from_prompt_to_another_cache(ctx, codec, layout, scaling):
    m, g = Model(ctx, layout, scaling), np.random.default_rng(int(codec))
    args = (LAYERS, KVH, HD, 16, 128, 16, 40, ROWS, int(codec))
    dev, ref = ctx.block_kv_cache(*args), bm.Cache(*args)
    mask = g.random(VOCAB) < 0.7
    m.bind(mask, 8000)
    text = {s: list(g.integers(0, VOCAB, n)) for s, n in enumerate((50, 17, 5))}

    def call(seqs, tokens, starts, eager=True):
        """The model over tokens[i] at starts[i] of seqs[i]; one history for each row."""
        counts = [len(t) for t in tokens]
        rows, history = sum(counts), []
        for s, a, n in zip(seqs, starts, counts):
            history += [text[s][:a + i + 1] for i in range(n)]
        print("[step]", seqs, starts, counts, flush=True)
        m.put(np.concatenate(tokens).astype(int), seqs, starts, counts, history)
        if eager:
            m.forward(dev, len(seqs), rows, max(counts), 128)
        else:
            eager_out = m.outputs(rows)
            graph.launch()
            ctx.synchronize()
            for a, b in zip(eager_out, m.outputs(rows)):
                assert np.array_equal(a, b)
        assert dev.status() == len(seqs)
        assert ref.step(list(seqs), list(starts), counts) == (bm.OK, len(seqs))
        m.compare(ref, rows, starts, counts, history, mask)
        return m.next.download(np.int32, rows)

    # the prompts in two chunks
    cut = {s: min(20, len(t)) for s, t in text.items()}
    call([0, 1, 2], [text[s][:cut[s]] for s in text], [0, 0, 0])
    nxt = call([0, 2], [text[0][cut[0]:], text[2][4:]], [cut[0], 4])  # the last row of prompt 2 once more
    # three candidates of each of two prompts
    live = [4, 5, 6, 7, 8, 9]
    parents = [0, 0, 0, 2, 2, 2]
    dev.fork(parents, live)
    assert ref.fork(parents, live)[0] == bm.OK
    last = {0: int(nxt[-2]), 2: int(nxt[-1])}
    for s, p in zip(live, parents):
        text[s] = text[p] + [int(g.integers(0, VOCAB)) if s % 2 else last[p]]
    graph = None
    for r in range(14):
        starts = [len(text[s]) - 1 for s in live]
        if r % 5 == 3:  # three drafted rows, of which one is kept: the next step takes two back
            drafts = [[text[s][-1]] + list(g.integers(0, VOCAB, 2)) for s in live]
            for s, d in zip(live, drafts):
                text[s] = text[s][:-1] + [int(t) for t in d]
            nxt = call(live, drafts, starts)[::3]
            for s in live:
                text[s] = text[s][:-2]
        else:
            nxt = call(live, [[text[s][-1]] for s in live], starts)
            if graph is None:
                graph = ctx.capture(lambda: m.forward(dev, 6, 6, 1, 128))
            # the same step again (its row is taken back), as a replay: bit for bit
            nxt = call(live, [[text[s][-1]] for s in live], starts, eager=False)
        assert np.all(nxt >= 0) and np.all(mask[nxt])
        for s, t in zip(live, nxt):
            text[s].append(int(t))
        if r % 3 == 2 and r % 5 != 3:  # the candidates' parents are chosen anew
            spare = [s for s in range(3, 16) if s not in live][:6]
            parents = [live[i] for i in np.r_[g.integers(0, 3, 3), 3 + g.integers(0, 3, 3)]]
            dev.fork(parents, spare)
            assert ref.fork(parents, spare)[0] == bm.OK
            dev.free(live)
            ref.free(live)
            for s, p in zip(spare, parents):
                text[s] = text[p][:-1] + [int(g.integers(0, VOCAB))]
            live = spare
        assert dev.pages()[0] == ref.free_pages()
    # one candidate of each prompt goes on in a smaller cache
    small = (LAYERS, KVH, HD, 3, 128, 16, 12, ROWS, int(codec))
    dev2, ref2 = ctx.block_kv_cache(*small), bm.Cache(*small)
    dev2.copy_from(dev, [live[5], live[0]], [0, 2])
    assert ref2.copy_from(ref, [live[5], live[0]], [0, 2])[0] == bm.OK
    text = {0: text[live[5]], 2: text[live[0]]}
    dev, ref = dev2, ref2
    for _ in range(3):
        nxt = call([2, 0], [[text[s][-1]] for s in (2, 0)], [len(text[s]) - 1 for s in (2, 0)])
        for s, t in zip((2, 0), nxt):
            text[s].append(int(t))
    dev.compact()
    ref.compact()
    call([0, 2], [[text[s][-1]] for s in (0, 2)], [len(text[s]) - 1 for s in (0, 2)])
