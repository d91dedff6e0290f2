"""A whole beam search over one layer's operators: prompts by head norms with rotation and packed causal attention,
steps by head norms, paged attention and packed attention to a memory, rules, selection and reordering. Run with
every step launched and with a captured step, and replayed without any reordering."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

from vokra_amd import hip

F = np.float32
D, HQ, HK, HD, V = 64, 4, 2, 64, 97
BEAMS, STEPS, END, EPS, BASE = 5, 9, 11, 1e-5, 10000.0
SCALE = HD ** -0.5
PROMPTS, MEMORY = np.array([1, 18, 7]), np.array([40, 1, 77])
G = len(PROMPTS)
N, MAX_TIME = G * BEAMS, 32


@pytest.fixture(scope="module")
def ctx():
    c = hip.HipContext(0)
    yield c
    c.close()


def weights():
    g = np.random.default_rng(3)
    r = lambda *s: g.standard_normal(s).astype(F)  # noqa: E731
    w = {"emb": r(V, D), "qk": r(D, (HQ + HK) * HD) / F(8), "v": r(D, HK * HD) / F(8), "out": r(HQ * HD, V) / F(8),
         "gq": 1 + r(HD) / F(4), "gk": 1 + r(HK, HD) / F(4), "mk": r(MEMORY.sum(), HK * HD),
         "mv": r(MEMORY.sum(), HK * HD), "prompt": g.integers(0, V, PROMPTS.sum())}
    allowed = g.random((G, V)) < 0.8
    allowed[:, END] = True
    w["allowed"] = np.repeat(allowed, BEAMS, 0)
    words = np.zeros((N, (V + 31) // 32), np.uint32)
    for v in range(V):
        words[:, v // 32] |= w["allowed"][:, v].astype(np.uint32) << np.uint32(v % 32)
    w["words"] = words
    return w


def off(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


class Search:
    """The layer's buffers; a step's inputs are the tokens' rows, the place and the beams' scores."""

    def __init__(self, ctx, w):
        self.ctx, self.w = ctx, w
        up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
        self.d = {k: up(w[k]) for k in ("qk", "v", "out", "gq", "gk", "mk", "mv", "words")}
        rows = max(N, int(PROMPTS.sum()))
        for name, width in (("x", D), ("pqk", (HQ + HK) * HD), ("q", HQ * HD), ("k", HK * HD), ("vv", HK * HD),
                            ("a", HQ * HD), ("c", HQ * HD), ("logits", V)):
            self.d[name] = up(np.zeros((rows, width), F))
        ids = lambda *s: up(np.zeros(s, np.int32))  # noqa: E731
        self.pos, self.lens, self.glens, self.parents, self.tokens, self.ended = (
            ids(rows), ids(N), ids(G), ids(G, BEAMS), ids(G, BEAMS), ids(G, BEAMS))
        self.scores, self.first = up(np.zeros((G, BEAMS), F)), up(np.zeros((G, V), F))
        self.zero = up(np.zeros(G, F))
        self.streams = up(np.arange(N, dtype=np.int32))
        self.prompt_off, self.mem_off, self.beam_off = up(off(PROMPTS)), up(off(MEMORY)), up(off([BEAMS] * G))
        self.rope = ctx.rope_plan(HD, 48, hip.RopeLayout.HALF, BASE)
        self.prompts = ctx.packed_attn(G, rows, rows, HQ, HK, HD)
        self.cross = ctx.packed_attn(G, rows, int(MEMORY.sum()), HQ, HK, HD)
        self.beams = ctx.beam_select(G, BEAMS, V, BEAMS)
        self.rules = hip.LogitsRules(n_bias=N, bias_ids=up(np.full(N, END, np.int32)), bias=up(np.full(N, 2.0, F)),
                                     bias_offsets=up(np.arange(N + 1, dtype=np.int32)), mask=self.d["words"],
                                     mask_stride=self.d["words"].nbytes // N // 4)  # some end
        self.kv = hip.KvCache(ctx, 1, HK, HD, N, MAX_TIME, 8)

    def project(self, n):
        d = self.d
        self.ctx.gemm_f32_dev(n, (HQ + HK) * HD, D, d["x"], d["qk"], d["pqk"])
        self.ctx.gemm_f32_dev(n, HK * HD, D, d["x"], d["v"], d["vv"])

    def normed(self, n):
        """q and k out of the projection's rows, each to rows of its own."""
        d, wide = self.d, (HQ + HK) * HD
        part = SimpleNamespace(ptr=C.c_void_p(d["pqk"].ptr.value + HQ * HD * 4))  # k's columns of the same rows
        self.rope.norm_apply_dev(n, self.pos, EPS, HQ, d["pqk"], d["gq"], d["q"], HK, part, d["gk"], d["k"],
                                 k_gamma_stride=HD, q_stride=wide, k_stride=wide, q_out_stride=HQ * HD,
                                 k_out_stride=HK * HD)

    def prefill(self, streams_of):
        """Prompts into the streams streams_of(group); the last rows' logits into `first`."""
        n, d = int(PROMPTS.sum()), self.d
        d["x"].upload(self.w["emb"][self.w["prompt"]])
        times = np.concatenate([np.arange(p) for p in PROMPTS]).astype(np.int32)
        self.pos.upload(times)
        self.project(n)
        self.normed(n)
        longest = int(PROMPTS.max())
        self.prompts.attn_dev(G, n, n, longest, longest, self.prompt_off, None, d["q"], d["k"], d["vv"], SCALE, d["a"],
                              causal=True)
        self.cross.attn_dev(G, n, int(MEMORY.sum()), longest, int(MEMORY.max()), self.prompt_off, self.mem_off, d["a"],
                            d["mk"], d["mv"], SCALE, d["c"])
        self.ctx.add_f32_dev(d["a"], d["c"], d["a"], n * HQ * HD)
        self.ctx.gemm_f32_dev(n, V, HQ * HD, d["a"], d["out"], d["logits"])
        k, v = d["k"].download(F, n * HK * HD).reshape(n, -1), d["vv"].download(F, n * HK * HD).reshape(n, -1)
        for g in range(G):
            i = slice(off(PROMPTS)[g], off(PROMPTS)[g + 1])
            for s in streams_of(g):
                self.kv.append(0, np.full(PROMPTS[g], s), times[i], k[i], v[i])
        all_logits = d["logits"].download(F, n * V).reshape(n, V)
        self.first.upload(all_logits[off(PROMPTS)[1:] - 1])
        return all_logits

    def place(self, tokens, step):
        at = np.repeat(PROMPTS + step, BEAMS).astype(np.int32)
        self.d["x"].upload(self.w["emb"][tokens.reshape(-1)])
        self.pos.upload(at)
        self.lens.upload(at + 1)
        self.glens.upload((PROMPTS + step + 1).astype(np.int32))

    def logits(self):
        d = self.d
        self.project(N)
        self.normed(N)
        self.kv.append_dev(0, N, self.streams, self.pos, d["k"], d["vv"])
        self.kv.attn_dev(0, N, self.streams, self.lens, MAX_TIME, HQ, d["q"], SCALE, d["a"])
        self.cross.attn_dev(G, N, int(MEMORY.sum()), BEAMS, int(MEMORY.max()), self.beam_off, self.mem_off, d["a"],
                            d["mk"], d["mv"], SCALE, d["c"])
        self.ctx.add_f32_dev(d["a"], d["c"], d["a"], N * HQ * HD)
        self.ctx.gemm_f32_dev(N, V, HQ * HD, d["a"], d["out"], d["logits"])
        self.ctx.logits_rules_dev(N, V, d["logits"], self.rules, d["logits"], None)

    def step(self):
        self.logits()
        self.beams.select_dev(G, BEAMS, V, BEAMS, self.d["logits"], self.scores, self.scores, self.parents, self.tokens,
                              d_ended=self.ended, end_token=END, d_out_ended=self.ended)
        self.kv.reorder_dev(G, BEAMS, self.streams, self.parents, self.glens, MAX_TIME)

    def got(self):
        i = [b.download(np.int32, N).reshape(G, BEAMS) for b in (self.parents, self.tokens, self.ended)]
        return (self.scores.download(F, N).reshape(G, BEAMS), *i)

    def run(self, captured):
        """[(scores, parents, tokens, ended, the step's logits or None)]: the first choice and the steps."""
        self.prefill(lambda g: [g * BEAMS])
        # every beam of a group goes on from the one that has read the prompt
        self.beams.select_dev(G, 1, V, BEAMS, self.first, self.zero, self.scores, self.parents, self.tokens,
                              end_token=END, d_out_ended=self.ended)
        self.glens.upload(PROMPTS.astype(np.int32))
        self.kv.reorder_dev(G, BEAMS, self.streams, self.parents, self.glens, MAX_TIME)
        out = [(*self.got(), None)]
        graph = None
        for step in range(STEPS):
            self.place(out[-1][2], step)
            if captured and step == 2:
                graph = self.ctx.capture(self.step)
            graph.launch() if graph else self.step()
            self.ctx.synchronize()
            out.append((*self.got(), self.d["logits"].download(F, N * V).reshape(G, BEAMS, V)))
        return out


def log_softmax(x):
    x = x.astype(np.float64)
    y = x - x.max(-1, keepdims=True)
    return y - np.log(np.exp(y).sum(-1, keepdims=True))


# a step's total against 64 bits: the sum of exponentials is f32 work of at most (3 * 2^7 + 1 + 32) roundings, and the
# score's own rounding on its way out
def step_tol(score):
    return 2.5e-5 + abs(score) * 2.0 ** -23


@pytest.fixture(scope="module")
def runs(ctx):
    w = weights()
    return w, Search(ctx, w).run(False), Search(ctx, w).run(True)


@pytest.mark.gpu
def test_prompts_against_64_bits(ctx):
    print("[case] beam search, prompts", flush=True)
    w = weights()
    got = Search(ctx, w).prefill(lambda g: [g])
    e = {k: (a.astype(np.float64) if a.dtype == F else a) for k, a in w.items()}
    x = e["emb"][w["prompt"]]
    qk, v = (x @ e["qk"]).reshape(len(x), HQ + HK, HD), (x @ e["v"]).reshape(len(x), HK, HD)
    gamma = np.concatenate([np.tile(e["gq"], (HQ, 1)), e["gk"]])
    qk = qk / np.sqrt((qk ** 2).mean(-1, keepdims=True) + EPS) * gamma
    pos = np.concatenate([np.arange(p) for p in PROMPTS])
    ang = pos[:, None, None] * BASE ** (-np.arange(24) / 24.0)
    a, b = qk[..., :24].copy(), qk[..., 24:48].copy()
    qk[..., :24], qk[..., 24:48] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)

    def attend(q, k, v, causal):
        q = q.reshape(len(q), HK, HQ // HK, HD)
        s = np.einsum("nkrd,mkd->krnm", q, k) * SCALE
        if causal:
            s = np.where(np.tri(len(k), dtype=bool), s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        o = np.einsum("krnm,mkd->nkrd", p / p.sum(-1, keepdims=True), v)
        return o.reshape(len(o), HQ * HD)
    mk, mv = e["mk"].reshape(-1, HK, HD), e["mv"].reshape(-1, HK, HD)
    po, mo = off(PROMPTS), off(MEMORY)
    for g in range(G):
        i, j = slice(po[g], po[g + 1]), slice(mo[g], mo[g + 1])
        o = attend(qk[i, :HQ], qk[i, HQ:], v[i], True)
        c = attend(o, mk[j], mv[j], False)
        want = (o + c) @ e["out"]
        # a projection's sums of 64: 2^-18 of |x| |w| at most; a normed head of 8 sqrt(gamma) in length, so scores of
        # up to some 2^5 off by 2^-12 at most (both sides 2^-18, their split 2^-21) and weights by as much of
        # themselves; the memory's scores take o's error times keys of up to 14 in length: 2^-11 in all, of rows of
        # V no larger than the largest, through the output's columns; roundings that do not all fall one
        # way leave the scores, and so the whole, within 2^5 * 2^-21 and the projections' 2^-21
        most = np.abs(v[i]).max() + np.abs(mv[j]).max()
        tol = 2.0 ** -11 * most * np.abs(e["out"]).sum(0)
        assert np.all(np.abs(got[i] - want) <= tol)
        assert np.linalg.norm(got[i] - want) <= 2.0 ** -15 * np.linalg.norm(want)


@pytest.mark.gpu
def test_a_captured_step_is_the_launched_one(runs):
    print("[case] beam search, captured", flush=True)
    for a, b in zip(runs[1], runs[2]):
        for x, y in zip(a, b):
            assert (x is None and y is None) or np.array_equal(x, y)


@pytest.mark.gpu
def test_every_selection(runs):
    """The totals that were taken are the largest, each its own."""
    print("[case] beam search, selections", flush=True)
    w, out, _ = runs
    old = None
    for scores, parents, tokens, ended, logits in out:
        if logits is not None:
            assert np.array_equal(np.isfinite(logits), w["allowed"].reshape(G, BEAMS, V))
            for g in range(G):
                total = old[0][g][:, None].astype(np.float64) + log_softmax(logits[g])
                for b in np.flatnonzero(old[3][g]):
                    total[b] = -np.inf
                    total[b, END] = old[0][g][b]
                taken = total[parents[g], tokens[g]]
                tol = np.array([step_tol(s) for s in taken])
                assert np.all(np.abs(taken - scores[g]) <= tol)
                assert np.all(np.diff(scores[g]) <= 0) and len(set(zip(parents[g], tokens[g]))) == BEAMS
                rest = total.copy()
                rest[parents[g], tokens[g]] = -np.inf
                assert rest.max() <= taken.min() + 2 * tol.max()
                assert np.array_equal(ended[g], (old[3][g][parents[g]] != 0) | (tokens[g] == END))
        old = scores, parents, tokens, ended
    assert old[3].any() and not old[3].all()  # hypotheses of both kinds


@pytest.mark.gpu
def test_hypotheses_read_from_scratch(ctx, runs):
    """Each hypothesis in a stream that read it itself, with no reordering, has the logits of every
    step bit for bit and its score."""
    print("[case] beam search, from scratch", flush=True)
    w, out, _ = runs
    path = [np.tile(np.arange(BEAMS), (G, 1))]  # which beam of each step a final one was
    for step in range(STEPS, 0, -1):
        path.append(np.take_along_axis(out[step][1], path[-1], 1))
    path = path[::-1]
    s = Search(ctx, w)
    s.prefill(lambda g: range(g * BEAMS, (g + 1) * BEAMS))
    first = log_softmax(s.first.download(F, G * V).reshape(G, V))
    total = np.take_along_axis(first, np.take_along_axis(out[0][2], path[0], 1), 1)
    over = np.take_along_axis(out[0][2], path[0], 1) == END
    tol = np.array([[step_tol(x) for x in r] for r in total])
    for step in range(STEPS):
        s.place(np.take_along_axis(out[step][2], path[step], 1), step)
        s.logits()
        s.ctx.synchronize()
        x = s.d["logits"].download(F, N * V).reshape(G, BEAMS, V)
        assert np.array_equal(x, np.take_along_axis(out[step + 1][4], path[step][..., None], 1)), step
        tok = np.take_along_axis(out[step + 1][2], path[step + 1], 1)
        total += np.where(over, 0, np.take_along_axis(log_softmax(x), tok[..., None], 2)[..., 0])
        over |= tok == END
        tol += np.array([[step_tol(v) for v in r] for r in total])
    assert np.all(np.abs(total - out[STEPS][0]) <= tol)
    assert np.array_equal(over, out[STEPS][3] != 0)
