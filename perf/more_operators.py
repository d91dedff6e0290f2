"""A prompt's pass without a cache, and a search of several beams, as timed cases on one GPU.

The operators: norms of q's and k's heads with their rotary positions in one
pass, attention over packed sequences of different lengths, beam search's
selection over beams and vocabulary, and the reordering of the paged Q8_0
cache's streams that follows it. With `own` set, `run` calls them through
vokra_amd.hip; without it, `run` computes the same from elementary torch
operations on plain tensors.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
_CTX = None


def _ctx():
    """The one device context a program holds."""
    global _CTX
    if _CTX is None:
        from vokra_amd import hip
        torch.cuda.init()
        _CTX = hip.HipContext(0)
    return _CTX


class _Dev:
    """A torch tensor (or the part of one from its first element on) as a device-pointer argument."""

    def __init__(self, t):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr())


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _i32(x):
    return _Dev(torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device=DEV))


def _spread(lo, hi, n):
    """n whole numbers spread evenly over lo..hi, ascending."""
    return np.round(np.linspace(lo, hi, n)).astype(np.int64)


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)])


# ---- family "norm": q and k of a fused projection's rows: each head by its root mean square and weights, turned

def _norm_inputs(c, seed):
    g = _gen(seed)
    hq, hk, hd, rows = c["heads"], c["kv_heads"], c["hd"], c["rows"]
    x = _randn(g, rows, (hq + 2 * hk) * hd)  # q, k and v side by side
    x *= torch.exp(0.5 * _randn(g, rows, 1))  # rows differ in size, and a few channels are large
    x *= 1.0 + 6.0 * (torch.rand(1, x.shape[1], generator=g, device=DEV) > 0.98)
    per = (lambda h: h) if c["per_head"] else (lambda h: 1)
    gq, gk = (1.0 + 0.2 * _randn(g, per(h), hd) for h in (hq, hk))
    # sequences one after another, each from its own position on
    run = min(c["run"], rows)
    first = torch.randint(0, c["pos_hi"], (-(-rows // run),), generator=g, device=DEV)
    pos = (first[:, None] + torch.arange(run, device=DEV)).reshape(-1)[:rows].to(torch.int32)
    return x, gq, gk, pos


def _norm_prepare(c, seed):
    x, gq, gk, pos = _norm_inputs(c, seed)
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    st = {"x": x, "gq": gq, "gk": gk, "pos": pos}
    if own:
        from vokra_amd import hip
        layout = hip.RopeLayout.HALF if c["layout"] == "half" else hip.RopeLayout.INTERLEAVED
        st["plan"] = _ctx().rope_plan(hd, c["rot"], layout, base=c["base"])
        st.update(q=_Dev(x), k=_Dev(x[:, hq * hd:]), d_gq=_Dev(gq), d_gk=_Dev(gk), d_pos=_Dev(pos),
                  qo=_Dev(torch.zeros(c["rows"], hq * hd, device=DEV)),
                  ko=_Dev(torch.zeros(c["rows"], hk * hd, device=DEV)))
        torch.cuda.synchronize()
    return st


def _turn(x, pos, c):
    """Heads [rows, h, hd] turned: cosines and sines of angles in 64 bits, as x's type."""
    rot = c["rot"]
    theta = float(c["base"]) ** (-2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot)
    a = pos.double()[:, None] * theta
    cos, sin = torch.cos(a).to(x.dtype)[:, None], torch.sin(a).to(x.dtype)[:, None]
    y = x.clone()
    if c["layout"] == "half":
        u, v = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        u, v = slice(0, rot, 2), slice(1, rot, 2)
    y[..., u] = x[..., u] * cos - x[..., v] * sin
    y[..., v] = x[..., u] * sin + x[..., v] * cos
    return y


def _norm_run(c, s):
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    if own:
        w = s["x"].shape[1]
        step = hd if c["per_head"] else 0
        s["plan"].norm_apply_dev(c["rows"], s["d_pos"], c["eps"], hq, s["q"], s["d_gq"], s["qo"], hk, s["k"], s["d_gk"],
                                 s["ko"], q_gamma_stride=step, k_gamma_stride=step, q_stride=w, k_stride=w)
        return [s["qo"].t, s["ko"].t]
    out = []
    for first, h, gamma in ((0, hq, s["gq"]), (hq, hk, s["gk"])):
        x = s["x"][:, first * hd:(first + h) * hd].reshape(-1, h, hd)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c["eps"]) * gamma
        out.append(_turn(y, s["pos"], c).reshape(-1, h * hd))
    return out


def _norm_exact(c, seed):
    x, gq, gk, pos = _norm_inputs(c, seed)
    hq, hk, hd, rot = c["heads"], c["kv_heads"], c["hd"], c["rot"]
    out = []
    for first, h, gamma in ((0, hq, gq), (hq, hk, gk)):
        y = x[:, first * hd:(first + h) * hd].double().reshape(-1, h, hd)
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + c["eps"]) * gamma.double()
        # the pairs as complex numbers
        p = y[..., :rot]
        z = torch.complex(*(p.unflatten(-1, (2, -1)).unbind(-2) if c["layout"] == "half"
                            else p.unflatten(-1, (-1, 2)).unbind(-1)))
        j = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
        a = pos.double()[:, None, None] * torch.exp(-2.0 * j / rot * math.log(c["base"]))
        z = z * torch.polar(torch.ones_like(a), a)
        p = torch.cat([z.real, z.imag], -1) if c["layout"] == "half" else torch.stack([z.real, z.imag], -1).flatten(-2)
        out.append(torch.cat([p, y[..., rot:]], -1).reshape(-1, h * hd))
    return out


def _norm_work(c):
    n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["hd"]
    return {"bytes": 8 * n + 4 * c["rows"], "flops": 7 * n}


# ---- family "attn": attention over packed sequences of different lengths, q, k and v parts of their rows

def _attn_shape(c, seed):
    """Rows of q and of k of every sequence, in an order of the seed's."""
    order = np.random.default_rng(int(seed)).permutation(c["seqs"])
    m = _spread(c["len_lo"], c["len_hi"], c["seqs"])
    n = m if not c["q_hi"] else np.roll(_spread(min(c["q_lo"], c["q_hi"]), c["q_hi"], c["seqs"]), c["seqs"] // 2)
    if c["causal"]:
        n = np.minimum(n, m)
    return n[order], m[order]


def _attn_inputs(c, seed):
    n, m = _attn_shape(c, seed)
    g = _gen(seed)
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    fused = not c["q_hi"]  # q, k and v of one projection
    x = _randn(g, int(m.sum()), ((hq if fused else 0) + 2 * hk) * hd)
    q = x[:, :hq * hd] if fused else _randn(g, int(n.sum()), hq * hd)
    k, v = (x[:, x.shape[1] - i * hk * hd:][:, :hk * hd] for i in (2, 1))
    k *= 1.0 + 3.0 * (torch.rand(1, hk * hd, generator=g, device=DEV) > 0.97)  # a few large channels, as keys have
    v *= 0.3 * torch.exp(0.5 * torch.sin(torch.arange(x.shape[0], device=DEV) / 37.0))[:, None]
    return n, m, q, k, v


def _attn_prepare(c, seed):
    n, m, q, k, v = _attn_inputs(c, seed)
    st = {"n": n, "m": m, "q": q, "k": k, "v": v}
    if own:
        st["plan"] = _ctx().packed_attn(c["seqs"], int(n.sum()), int(m.sum()), c["heads"], c["kv_heads"], c["hd"])
        st.update(d_q=_Dev(q), d_k=_Dev(k), d_v=_Dev(v), n_off=_i32(_offsets(n)), m_off=_i32(_offsets(m)),
                  out=_Dev(torch.zeros(int(n.sum()), c["heads"] * c["hd"], device=DEV)))
        torch.cuda.synchronize()
    return st


def _seen(c, a, b, n, m):
    """Which of m keys the rows a..b of n see: the last row sees the last key."""
    p = torch.arange(a, b, device=DEV)[:, None] + (m - n)
    j = torch.arange(m, device=DEV)[None]
    seen = j <= p
    return seen & (j > p - c["window"]) if c["window"] else seen


def _attn_run(c, s):
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    n, m = s["n"], s["m"]
    if own:
        s["plan"].attn_dev(c["seqs"], int(n.sum()), int(m.sum()), int(n.max()), int(m.max()), s["n_off"], s["m_off"],
                           s["d_q"], s["d_k"], s["d_v"], hd ** -0.5, s["out"], causal=c["causal"], window=c["window"],
                           q_stride=s["q"].stride(0), k_stride=s["k"].stride(0), v_stride=s["v"].stride(0))
        return s["out"].t
    out = torch.empty(int(n.sum()), hq, hd, device=DEV)
    an, am, r = _offsets(n), _offsets(m), hq // hk
    for i in range(c["seqs"]):
        k, v = (s[x][int(am[i]):int(am[i + 1])].reshape(-1, hk, hd).transpose(0, 1).contiguous() for x in "kv")
        q = s["q"][int(an[i]):int(an[i + 1])].reshape(-1, hk, r, hd) * hd ** -0.5
        for a in range(0, int(n[i]), 512):
            b = min(int(n[i]), a + 512)
            x = torch.matmul(q[a:b].permute(1, 2, 0, 3).reshape(hk, r * (b - a), hd), k.transpose(1, 2).contiguous())
            if c["causal"]:
                seen = _seen(c, a, b, int(n[i]), int(m[i])).repeat(r, 1)
                x = x.masked_fill(~seen, -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            y = torch.matmul(x, v) / x.sum(-1, keepdim=True)
            out[int(an[i]) + a:int(an[i]) + b] = y.reshape(hk, r, b - a, hd).permute(2, 0, 1, 3).reshape(b - a, hq, hd)
    return out.reshape(-1, hq * hd)


def _attn_exact(c, seed):
    n, m, q, k, v = _attn_inputs(c, seed)
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    out = torch.empty(q.shape[0], hq, hd, dtype=torch.float64, device=DEV)
    an, am = _offsets(n), _offsets(m)
    for i in range(c["seqs"]):
        for h in range(hq):
            kv = h // (hq // hk)
            kk, vv = (x[int(am[i]):int(am[i + 1]), kv * hd:(kv + 1) * hd].double() for x in (k, v))
            qq = q[int(an[i]):int(an[i + 1]), h * hd:(h + 1) * hd].double()
            for a in range(0, int(n[i]), 2048):
                b = min(int(n[i]), a + 2048)
                x = qq[a:b] @ kk.T.contiguous() / math.sqrt(hd)
                if c["causal"]:
                    x[~_seen(c, a, b, int(n[i]), int(m[i]))] = -math.inf
                out[int(an[i]) + a:int(an[i]) + b, h] = torch.softmax(x, -1) @ vv
    return out.reshape(-1, hq * hd)


def _attn_work(c):
    n, m = _attn_shape(c, 0)
    pairs = 0
    for a, b in zip(n, m):
        if not c["causal"]:
            pairs += int(a * b)
            continue
        p = np.arange(b - a, b)
        pairs += int((np.minimum(p + 1, c["window"]) if c["window"] else p + 1).sum())
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    return {"bytes": 4 * hd * (2 * hq * int(n.sum()) + 2 * hk * int(m.sum())), "flops": 4 * hq * hd * pairs}


# ---- family "select": the best continuations of every group's beams

def _select_inputs(c, seed):
    g = _gen(seed)
    rows = c["groups"] * c["beams"]
    x = 2.0 * _randn(g, rows, c["vocab"])
    # a few tokens stand out in each row, as a model's do, and rules have struck some out
    top = torch.randint(0, c["vocab"], (rows, 24), generator=g, device=DEV)
    x.scatter_(1, top, 9.0 + 2.0 * _randn(g, rows, 24))
    if c["struck"]:
        x[torch.rand(rows, c["vocab"], generator=g, device=DEV) < c["struck"]] = -math.inf
    scores = -3.0 * torch.rand(rows, generator=g, device=DEV) - 0.5 * torch.arange(c["beams"], device=DEV).repeat(
        c["groups"])
    ended = (torch.rand(rows, generator=g, device=DEV) < c["ended"]).to(torch.int32)
    return x, scores, ended


def _select_prepare(c, seed):
    x, scores, ended = _select_inputs(c, seed)
    st = {"x": x, "scores": scores, "ended": ended}
    if own:
        n = c["groups"] * c["n_out"]
        st["plan"] = _ctx().beam_select(c["groups"], c["beams"], c["vocab"], c["n_out"])
        st.update(d_x=_Dev(x), d_scores=_Dev(scores), d_ended=_Dev(ended),
                  out=[_Dev(torch.zeros(n, device=DEV, dtype=t)) for t in (torch.float32,) + 3 * (torch.int32,)])
        torch.cuda.synchronize()
    return st


def _end_token(c):
    return c["vocab"] - 1


def _select_run(c, s):
    g, b, v, n = c["groups"], c["beams"], c["vocab"], c["n_out"]
    if own:
        o = s["out"]
        s["plan"].select_dev(g, b, v, n, s["d_x"], s["d_scores"], *o[:3], d_ended=s["d_ended"], end_token=_end_token(c),
                             d_out_ended=o[3])
        return [x.t for x in o]
    # totals in 64 bits: continuations of different beams may be next to each other
    x = s["x"].double()
    top = x.amax(-1, keepdim=True)
    x = x - top
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    x = s["scores"].double()[:, None] + x
    ended = s["ended"].bool()
    x[ended] = -math.inf
    x[ended, _end_token(c)] = s["scores"].double()[ended]
    # of equal totals the lower index stands first
    val, at = torch.sort(x.reshape(g, b * v), dim=-1, descending=True, stable=True)
    val, at = val[:, :n], at[:, :n]
    parents, tokens = at // v, at % v
    over = torch.gather(s["ended"].reshape(g, b), 1, parents) | (tokens == _end_token(c)).to(torch.int32)
    none = val == -math.inf  # fewer continuations than asked for
    parents, tokens, over = parents.masked_fill(none, -1), tokens.masked_fill(none, -1), over.masked_fill(none, 1)
    return [val.float().reshape(-1), parents.to(torch.int32).reshape(-1), tokens.to(torch.int32).reshape(-1),
            over.to(torch.int32).reshape(-1)]


def _select_exact(c, seed):
    x, scores, ended = _select_inputs(c, seed)
    g, b, v, n = c["groups"], c["beams"], c["vocab"], c["n_out"]
    keep = min(v, n + 8)
    out = [[], [], [], []]
    # each row's best by themselves, then each group's in numpy
    best, at = torch.topk(x, keep, dim=-1)
    lse = torch.logsumexp(x.double(), -1).cpu().numpy()
    best, at, scores, ended = best.double().cpu().numpy(), at.cpu().numpy(), scores.double().cpu().numpy(), ended.cpu().numpy()
    for i in range(g):
        tot, par, tok = [], [], []
        for j in range(b):
            r = i * b + j
            if ended[r]:
                tot.append(scores[r:r + 1]), par.append([j]), tok.append([_end_token(c)])
            else:
                tot.append(scores[r] + (best[r] - lse[r])), par.append(np.full(keep, j)), tok.append(at[r])
        tot, par, tok = (np.concatenate(z) for z in (tot, par, tok))
        first = np.lexsort((tok, par, -tot))
        first = first[tot[first] > -np.inf][:n]
        over = ended.reshape(g, b)[i][par[first]].astype(bool) | (tok[first] == _end_token(c))
        for o, z, rest in zip(out, (tot[first], par[first], tok[first], over), (-np.inf, -1, -1, 1)):
            o.append(np.concatenate([z, np.full(n - first.size, rest)]))
    types = (torch.float64,) + 3 * (torch.int32,)
    return [torch.as_tensor(np.concatenate(z)).to(t).to(DEV) for z, t in zip(out, types)]


def _select_work(c):
    rows = c["groups"] * c["beams"]
    return {"bytes": 4 * rows * (c["vocab"] + 2) + 16 * c["groups"] * c["n_out"], "flops": 4 * rows * c["vocab"]}


# ---- family "reorder": the paged Q8_0 cache's streams after a selection, every layer, and the attention of the
# step that follows, every layer in turn

def _reorder_inputs(c, seed):
    rng = np.random.default_rng(int(seed))
    g, b = c["groups"], c["beams"]
    lens = rng.permutation(_spread(c["len_lo"], c["len_hi"], g))
    # beams that go on keep their places, each of the others takes one of those
    parents = np.empty((g, b), np.int64)
    for i in range(g):
        stay = np.sort(rng.choice(b, max(1, b - max(1, int(b * c["moved"]))), replace=False))
        parents[i] = rng.choice(stay, b)
        parents[i][stay] = stay
    streams = rng.permutation(g * b).reshape(g, b)
    gen = _gen(seed)
    rows = [[_randn(gen, g * b, int(lens.max()), c["kv_heads"], c["hd"]) for _ in (0, 1)] for _ in range(c["layers"])]
    q = _randn(gen, c["layers"], g * b, c["heads"] * c["hd"])
    return lens, parents, streams, rows, q


def _pack_q8(x):
    """Blocks of 32 under an f16 scale: (values, scales as f32)."""
    y = x.unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    d = torch.div(a, torch.full_like(a, 127.0))
    z = y * torch.div(torch.ones_like(d), d)
    t = torch.trunc(z)
    t = t + torch.sign(z) * ((z - t).abs() >= 0.5)  # halves away from zero
    return t.clamp(-127.0, 127.0).to(torch.int8), d.half().float()


def _reorder_prepare(c, seed):
    lens, parents, streams, rows, q = _reorder_inputs(c, seed)
    g, b, n = c["groups"], c["beams"], c["groups"] * c["beams"]
    st = {"lens": lens, "parents": parents, "q": q}
    if not own:
        st["packed"] = [[_pack_q8(x) for x in sides] for sides in rows]
        return st
    from vokra_amd import hip
    most = int(lens.max())
    kv = hip.KvCache(_ctx(), c["layers"], c["kv_heads"], c["hd"], n, most, c["bs"])
    row_len = np.repeat(lens, b)  # of beam i of a group
    item = np.repeat(np.arange(n), row_len)
    time = np.concatenate([np.arange(t) for t in row_len])
    for a in range(0, item.size, 1024):
        i, t = item[a:a + 1024], time[a:a + 1024]
        d_s, d_t = _i32(streams.reshape(-1)[i]), _i32(t)
        for layer in range(c["layers"]):
            k, v = (_Dev(x[i, t].contiguous()) for x in rows[layer])
            torch.cuda.synchronize()
            kv.append_dev(layer, i.size, d_s, d_t, k, v)
            _ctx().synchronize()
    st.update(kv=kv, streams=_i32(streams.reshape(-1)), d_parents=_i32(parents.reshape(-1)), d_lens=_i32(lens),
              row_len=_i32(row_len), d_q=[_Dev(x) for x in q], out=[_Dev(torch.zeros_like(x)) for x in q])
    torch.cuda.synchronize()
    return st


def _reorder_run(c, s):
    g, b, n = c["groups"], c["beams"], c["groups"] * c["beams"]
    hq, hk, hd = c["heads"], c["kv_heads"], c["hd"]
    most = int(s["lens"].max())
    if own:
        kv = s["kv"]
        kv.reorder_dev(g, b, s["streams"], s["d_parents"], s["d_lens"], most)
        for layer in range(c["layers"]):
            kv.attn_dev(layer, n, s["streams"], s["row_len"], most, hq, s["d_q"][layer], hd ** -0.5, s["out"][layer])
        return [o.t for o in s["out"]]
    src = torch.as_tensor((np.arange(g)[:, None] * b + s["parents"]).reshape(-1), device=DEV)
    lens = torch.as_tensor(np.repeat(s["lens"], b), device=DEV)
    gone = torch.arange(most, device=DEV)[None] >= lens[:, None]
    out = []
    for layer in range(c["layers"]):
        k, v = ((z[src].float() * d[src]).flatten(-2).transpose(1, 2).contiguous() for z, d in s["packed"][layer])
        q = s["q"][layer].reshape(n, hk, hq // hk, hd) * hd ** -0.5
        x = torch.matmul(q, k.transpose(2, 3).contiguous()).masked_fill(gone[:, None, None], -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        out.append((torch.matmul(x, v) / x.sum(-1, keepdim=True)).reshape(n, hq * hd))
    return out


def _reorder_exact(c, seed):
    lens, parents, _, rows, q = _reorder_inputs(c, seed)
    hq, hk, hd, b = c["heads"], c["kv_heads"], c["hd"], c["beams"]
    out = []
    for layer in range(c["layers"]):
        y = torch.empty(q.shape[1], hq, hd, dtype=torch.float64, device=DEV)
        sides = [_pack_q8(x) for x in rows[layer]]
        for i, p in enumerate(parents.reshape(-1)):
            at, t = i // b * b + int(p), int(lens[i // b])
            k, v = ((z[at, :t].double() * d[at, :t].double()).flatten(-2) for z, d in sides)
            x = q[layer, i].double().reshape(hk, hq // hk, hd) @ k.permute(1, 2, 0).contiguous() / math.sqrt(hd)
            y[i] = (torch.softmax(x, -1) @ v.transpose(0, 1).contiguous()).reshape(hq, hd)
        out.append(y.reshape(-1, hq * hd))
    return out


def _reorder_work(c):
    g, b, w = c["groups"], c["beams"], c["kv_heads"] * c["hd"]
    lens = _spread(c["len_lo"], c["len_hi"], g)
    row = 2 * (w + w // 32 * 2)  # bytes of K and V of a position as the cache holds them
    moved = max(1, int(b * c["moved"])) if b > 1 else 0  # written; at least one stream of a group is read for them
    n = int(lens.sum())
    return {"bytes": c["layers"] * (n * row * (moved + (1 if moved else 0) + b) + 8 * g * b * c["heads"] * c["hd"]),
            "flops": 4 * c["layers"] * c["heads"] * c["hd"] * b * n}


_FAMILY = {
    "norm": (_norm_prepare, _norm_run, _norm_exact, _norm_work),
    "attn": (_attn_prepare, _attn_run, _attn_exact, _attn_work),
    "select": (_select_prepare, _select_run, _select_exact, _select_work),
    "reorder": (_reorder_prepare, _reorder_run, _reorder_exact, _reorder_work),
}


def _case(family, **kw):
    return dict(family=family, **kw)


def listed():
    attn = dict(q_lo=0, q_hi=0, causal=True, window=0)
    return [
        # one token of each of 32 streams of the text decoder (16 heads over 2 of 128), behind its q/k/v projection
        _case("norm", name="norm_step", heads=16, kv_heads=2, hd=128, rot=128, layout="half", base=1e6, eps=1e-5,
              rows=32, run=1, pos_hi=4096, per_head=False),
        # prompts of 700 rows, packed, of a larger decoder
        _case("norm", name="norm_prompts", heads=32, kv_heads=8, hd=128, rot=128, layout="half", base=1e6, eps=1e-5,
              rows=8191, run=700, pos_hi=30000, per_head=False),
        # three commands of a few words each: what a call costs
        _case("attn", name="attn_commands", heads=16, kv_heads=2, hd=128, seqs=3, len_lo=5, len_hi=61, **attn),
        # the prompts that a text decoder takes in at once, from a line to a page
        _case("attn", name="attn_prompts", heads=16, kv_heads=2, hd=128, seqs=16, len_lo=33, len_hi=2047, **attn),
        # utterances of 2 to 30 seconds through an encoder's attention, each against itself
        _case("attn", name="attn_utterances", heads=20, kv_heads=20, hd=64, seqs=8, len_lo=97, len_hi=1500,
              **{**attn, "causal": False}),
        # two long documents
        _case("attn", name="attn_documents", heads=32, kv_heads=8, hd=128, seqs=2, len_lo=5001, len_hi=8192, **attn),
        # a step of five candidates for each of 16 utterances, against the rows of its encoder
        _case("attn", name="attn_cross_step", heads=20, kv_heads=20, hd=64, seqs=16, len_lo=97, len_hi=1500, q_lo=5,
              q_hi=5, causal=False, window=0),
        # five beams of one utterance, the ten best continuations
        _case("select", name="select_utterance", groups=1, beams=5, vocab=51865, n_out=10, struck=0.0, ended=0.0),
        # 64 utterances at once, rules have struck tokens out, some beams have ended
        _case("select", name="select_streams", groups=64, beams=5, vocab=51866, n_out=5, struck=0.2, ended=0.15),
        # a text decoder's large vocabulary, eight beams, sixteen continuations
        _case("select", name="select_large", groups=32, beams=8, vocab=128259, n_out=16, struck=0.0, ended=0.1),
        # five beams of one prompt of a text decoder
        _case("reorder", name="reorder_prompt", heads=16, kv_heads=2, hd=128, bs=16, layers=4, groups=1, beams=5,
              len_lo=301, len_hi=301, moved=0.4),
        # twelve utterances of five beams each near the end of their texts
        _case("reorder", name="reorder_streams", heads=20, kv_heads=20, hd=64, bs=16, layers=8, groups=12, beams=5,
              len_lo=100, len_hi=447, moved=0.4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["norm", "attn", "attn", "attn", "select", "select", "reorder"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 20])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8] if kv_heads < 8 else [1, 4] if kv_heads < 20 else [1])
    hd = rng.choice([64, 128])
    if family == "norm":
        hd = rng.choice([64, 80, 96, 128, 256])
        rot = max(4, rng.choice([hd, hd, hd // 2, hd // 4, rng.randint(2, hd // 2) * 2]) // 2 * 2)
        most = int(4e7 / ((heads + 2 * kv_heads) * hd))
        return _case("norm", heads=heads, kv_heads=kv_heads, hd=hd, rot=rot, layout=rng.choice(["half", "pairs"]),
                     base=rng.choice([10000.0, 500000.0, 1e6]), eps=rng.choice([1e-5, 1e-6]),
                     rows=_log(rng, 1, min(8000, most)), run=rng.choice([1, 7, 500]),
                     pos_hi=_log(rng, 600, 100000), per_head=rng.random() < 0.4)
    if family == "attn":
        how = rng.choice(["prompts", "prompts", "context", "utterances", "step"])
        seqs = _log(rng, 1, 48)
        if how == "step":  # tokens or candidates against rows of their own
            most = 6e7 / (seqs * kv_heads * hd)
            hi = _log(rng, 2, max(2, min(16000, int(most))))
            n = rng.randint(1, max(1, 32 // (heads // kv_heads)))
            causal = n == 1 and rng.random() < 0.5
            return _case("attn", heads=heads, kv_heads=kv_heads, hd=hd, seqs=seqs, len_lo=rng.randint(1, hi), len_hi=hi,
                         q_lo=n if causal else rng.randint(1, n), q_hi=n, causal=causal, window=0)
        # (a sequence of its longest has pairs of at most about the largest listed case's)
        most = math.sqrt(4e11 / (4 * heads * hd * seqs))
        hi = _log(rng, 4, max(4, min(8000, int(most))))
        n = rng.randint(1, hi) if how == "context" else 0
        causal = how != "utterances"
        return _case("attn", heads=heads, kv_heads=kv_heads, hd=hd, seqs=seqs, len_lo=rng.randint(1, hi), len_hi=hi,
                     q_lo=rng.randint(1, n) if n else 0, q_hi=n, causal=causal,
                     window=_log(rng, 1, hi) if causal and rng.random() < 0.35 else 0)
    if family == "select":
        beams = rng.randint(1, 12)
        vocab = _log(rng, 1000, 150000)
        return _case("select", groups=_log(rng, 1, max(1, min(64, int(2.5e7 / (vocab * beams))))), beams=beams, vocab=vocab,
                     n_out=rng.choice([beams, 2 * beams]), struck=rng.choice([0.0, 0.0, 0.3]),
                     ended=rng.choice([0.0, 0.2]))
    beams, layers = rng.randint(2, 8), rng.randint(1, 6)
    r = rng.choice([1, 2, 4, 8])
    groups = _log(rng, 1, 12)
    hi = _log(rng, 3, max(3, min(448, int(2.5e7 / (groups * beams * layers * kv_heads * hd)))))
    return _case("reorder", heads=kv_heads * r, kv_heads=kv_heads, hd=hd, bs=rng.choice([16, 32, 64]), layers=layers,
                 groups=groups, beams=beams, len_lo=rng.randint(1, hi), len_hi=hi, moved=rng.choice([0.2, 0.5, 0.8]))


def prepare(case, seed):
    c = dict(case)
    state = _FAMILY[c["family"]][0](c, seed)
    state["case"] = c
    return state


def run(state):
    c = state["case"]
    return _FAMILY[c["family"]][1](c, state)


def exact(case, seed):
    return _FAMILY[case["family"]][2](dict(case), seed)


def work(case):
    return _FAMILY[case["family"]][3](dict(case))
