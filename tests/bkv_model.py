"""The block-scaled KV cache restated with numpy: rounding, planning (pages,
lengths, take-backs, forks, frees, copies, compaction) and attention in 64 bits."""
import numpy as np

OK, INVALID, EXHAUSTED = 0, 5, 10
TOP = {0: np.float32(127.0), 1: np.float32(448.0)}  # KvCodec -> largest value


def e4m3(y):
    """The nearest OCP e4m3 value of y (f32, |y| < 464), ties to even: the values
    have 3 mantissa bits from 2^-6 up and steps of 2^-9 below."""
    y = np.asarray(y, np.float64)
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(np.abs(y)))
    step = np.exp2(np.maximum(e, -6.0) - 3.0)
    return np.clip(np.rint(y / step) * step, -448.0, 448.0).astype(np.float32)


def held_block(x, codec):
    """The values a full block [bs, heads, hd] (f32) is held as."""
    x = np.asarray(x, np.float32)
    out = np.empty_like(x)
    for h in range(x.shape[1]):
        b = x[:, h]
        if not np.all(np.isfinite(b)):
            out[:, h] = np.nan
            continue
        a = np.abs(b).max().astype(np.float32)
        if a < np.float32(2.0 ** -100):
            out[:, h] = 0.0
            continue
        y = b * (TOP[codec] / a)
        q = np.rint(y) if codec == 0 else e4m3(y)
        out[:, h] = q.astype(np.float32) * (a / TOP[codec])
    return out


class Cache:
    """One cache; rows are kept as they came, per layer and side."""

    def __init__(self, n_layer, n_head, d_head, n_seq, max_time, bs, n_page, max_rows, codec=0):
        self.n_layer, self.n_head, self.hd, self.bs = n_layer, n_head, d_head, bs
        self.n_seq, self.max_time, self.n_page, self.max_rows, self.codec = n_seq, max_time, n_page, max_rows, codec
        self.reset()

    def reset(self):
        self.len = [0] * self.n_seq
        self.floor = [0] * self.n_seq
        self.table = [[] for _ in range(self.n_seq)]
        self.refs = [0] * self.n_page
        self.rows = [np.zeros((self.n_layer, 2, 0, self.n_head, self.hd), np.float32) for _ in range(self.n_seq)]
        self.plan = []

    def free_pages(self):
        return self.refs.count(0)

    def _take(self, n, avoid):
        got = [p for p in range(self.n_page) if self.refs[p] == 0 and p not in avoid][:n]
        for p in got:
            self.refs[p] = 1
        return got

    def _drop(self, page):
        self.refs[page] -= 1

    def step(self, seqs, starts, counts, n_rows=None, max_count=None):
        """(status, items done)"""
        bs, row0, free, named = self.bs, 0, self.free_pages(), set()
        self.plan, status, dropped = [], OK, []
        for s, a, n in zip(seqs, starts, counts):
            if not (0 <= s < self.n_seq) or s in named or n < 0 or a < self.floor[s] or a > self.len[s] or \
                    a + n > self.max_time or (max_count is not None and n > max_count) or \
                    (n_rows is not None and row0 + n > n_rows):
                status = INVALID
                break
            need = (a + n) // bs - a // bs
            if need > free:
                status = EXHAUSTED
                break
            free -= need
            named.add(s)
            self.plan.append((s, a, n, row0))
            row0 += n
        # every page of the call is taken before any is given up
        taken = [self._take((a + n) // bs - a // bs, ()) for _, a, n, _ in self.plan]
        for (s, a, n, _), pages in zip(self.plan, taken):
            dropped += self.table[s][a // bs:]
            self.table[s] = self.table[s][:a // bs] + pages
            self.len[s] = a + n
            self.floor[s] = max(self.floor[s], (-(-(a + n) // bs) - 2) * bs)
            x = self.rows[s][:, :, :a]
            self.rows[s] = np.concatenate([x, np.zeros((*x.shape[:2], n, *x.shape[3:]), np.float32)], 2)
        for p in dropped:
            self._drop(p)
        return status, len(self.plan)

    def write(self, layer, k, v):
        for s, a, n, r in self.plan:
            for side, x in ((0, k), (1, v)):
                self.rows[s][layer, side, a:a + n] = np.asarray(x).reshape(-1, self.n_head, self.hd)[r:r + n]

    def _pairs(self, src_cache, src, dst):
        named, good = set(), []
        for s, d in zip(src, dst):
            bad = not (0 <= s < src_cache.n_seq) or not (0 <= d < self.n_seq) or d in named or self.len[d] != 0 or \
                (src_cache is self and s in dst)
            if bad:
                return INVALID, good
            named.add(d)
            good.append((s, d))
        return OK, good

    def fork(self, src, dst):
        status, pairs = self._pairs(self, list(src), list(dst))
        for s, d in pairs:
            self.len[d], self.table[d], self.rows[d] = self.len[s], list(self.table[s]), self.rows[s].copy()
            self.floor[d] = max(self.floor[s], self.len[s] // self.bs * self.bs)
            for p in self.table[d]:
                self.refs[p] += 1
        return status, len(pairs)

    def free(self, seqs):
        self.plan = []
        for i, s in enumerate(seqs):
            if not 0 <= s < self.n_seq:
                return INVALID, i
            for p in self.table[s]:
                self._drop(p)
            self.len[s], self.floor[s], self.table[s] = 0, 0, []
            self.rows[s] = self.rows[s][:, :, :0]
        return OK, len(seqs)

    def copy_from(self, other, src, dst):
        status, pairs = self._pairs(other, list(src), list(dst))
        for i, (s, d) in enumerate(pairs):
            if other.len[s] > self.max_time:
                return INVALID, i
            if len(other.table[s]) > self.free_pages():
                return EXHAUSTED, i
            self.len[d], self.floor[d], self.rows[d] = other.len[s], other.floor[s], other.rows[s].copy()
            self.table[d] = self._take(len(other.table[s]), ())
        return status, len(pairs)

    def compact(self):
        u = self.n_page - self.free_pages()
        holes = [p for p in range(u) if self.refs[p] == 0]
        movers = [p for p in range(u, self.n_page) if self.refs[p]]
        to = dict(zip(movers, holes))
        for p, h in to.items():
            self.refs[h], self.refs[p] = self.refs[p], 0
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return OK, len(movers)

    def held(self, layer, s):
        """(K, V) of a sequence as the cache holds them, [len, heads, hd]."""
        out = []
        for side in (0, 1):
            x = self.rows[s][layer, side].copy()
            for b in range(self.len[s] // self.bs):
                r = slice(b * self.bs, (b + 1) * self.bs)
                x[r] = held_block(x[r], self.codec)
            out.append(x)
        return out

    def attn(self, layer, q, n_head_q, scale):
        """(out, bound) of the current step's rows in 64 bits, [rows, n_head_q * hd]:
        see attention for the bound. Rows outside the step are NaN."""
        q = np.asarray(q, np.float64).reshape(-1, n_head_q, self.hd)
        out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
        for s, a, n, r in self.plan:
            k, v = self.held(layer, s)
            reach = np.abs(np.asarray(v, np.float64)).max(2)  # [rows, kv heads], then of the row's block
            for b in range(0, len(reach), self.bs):
                reach[b:b + self.bs] = reach[b:b + self.bs].max(0)
            out[r:r + n], tol[r:r + n] = attention(q[r:r + n], k[:a + n], v[:a + n], a, scale, reach)
        return out.reshape(len(q), -1), tol.reshape(len(q), -1)


def attention(q, k, v, first, scale, reach):
    """Causal attention of q [n, heads, hd] at positions first.. over k, v [t, kv_heads, hd]
    in 64 bits, and a bound on the error of a correct f32 evaluation:
    a score is a sum of hd products of operands held to 2^-22, scaled to base 2
    (a few more roundings), so it is off by at most ds = (2^-22 + (hd + 8) 2^-24)
    scale |q| . |k|; weights are then off by a factor e^(2 ds) and the roundings
    of exp2 and of their two-part form (2^-21 together); sums over t keys add
    t 2^-24; all relative to sum p |v|.
    Two fp16 parts hold their operand to 2^-22 down to the end of fp16's range
    only. q's row is scaled so that its largest value is 2^14 at least, half of
    fp16's smallest step is 2^-25: 2^-39 of that largest value for every
    element, so ds grows by 2^-39 scale max|q| sum|k|. A weight w = p 2^e of the
    largest 2^M = max p 2^e is held as 2^14 w 2^-M: off by 2^-39 2^M, times a
    stored value of at most top (127 or 448) where 2^e top <= a, the largest
    magnitude of the block (`reach`): 2^-39 max(p a) for each of the t keys."""
    n, heads, hd = q.shape
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    rep = heads // k.shape[1]
    out, tol = np.empty((n, heads, hd)), np.empty((n, heads, hd))
    t = np.arange(len(k))
    for h in range(heads):
        kh, vh = k[:, h // rep], v[:, h // rep]
        for i in range(n):
            m = first + i + 1
            sc = kh[:m] @ q[i, h] * scale
            p = np.exp(sc - sc.max())
            p /= p.sum()
            out[i, h] = p @ vh[:m]
            ds = (2.0 ** -22 + (hd + 8) * 2.0 ** -24) * abs(scale) * (np.abs(kh[:m]) @ np.abs(q[i, h])).max()
            ds += 2.0 ** -39 * abs(scale) * np.abs(q[i, h]).max() * np.abs(kh[:m]).sum(1).max()
            tol[i, h] = (2 * ds + 2.0 ** -21 + (m + 8) * 2.0 ** -24) * (p @ np.abs(vh[:m])) + 1e-37
            tol[i, h] += m * 2.0 ** -39 * (p * reach[:m, h // rep]).max()
    return out, tol
