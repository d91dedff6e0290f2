"""The block-scaled KV cache and what a generation step does around it, as timed cases on one GPU.

The operators: rotary positions of q and k, the write into a paged cache held
in 8 bits (one scale for each block of tokens, head and side), attention over
it, the forking / copying / compacting / freeing of its pages, and the rules
(penalties, biases, grammar masks) that logits pass before the greedy choice.
With `own` set, `run` calls them through vokra_amd.hip; without it, `run`
computes the same from elementary torch operations on plain tensors.

The cache as both sides define it: rows of a sequence fall into blocks of
`bs` tokens. A full block holds, per head, 8-bit values under one f32 scale;
with a = max |x| over the block (all f32 operations, each rounded once):
int8: scale a / 127, value rint(x * (127 / a)); e4m3: scale a / 448, value
e4m3(x * (448 / a)). The rows of the last block, while it is not full, are held
as they came.
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
    """A torch tensor as the device-pointer argument of a resident call."""

    def __init__(self, t):
        assert t.is_contiguous()
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


def _div(a, b):
    """a / b rounded once (a division by a Python number may become a product)."""
    return torch.div(a, torch.full_like(a, b))


# ---- the cache's rounding, plain and in 64 bits ------------------------------

_TOP = {"int8": 127.0, "e4m3": 448.0}


def _pack(x, codec):
    """x [blocks, bs, heads, hd] f32 -> (8-bit values, scales [blocks, 1, heads, 1])."""
    a = x.abs().amax((1, 3), keepdim=True)
    small = a < 2.0 ** -100
    top = _TOP[codec]
    safe = torch.where(small, torch.ones_like(a), a)
    y = x * torch.div(torch.full_like(a, top), safe)
    y = torch.where(small, torch.zeros_like(y), y)
    q = torch.round(y).to(torch.int8) if codec == "int8" else y.to(torch.float8_e4m3fn)
    return q, torch.where(small, torch.zeros_like(a), _div(a, top))


def _held(x, codec, bs):
    """The values a cache holds for the rows x [t, heads, hd] (f32)."""
    n = x.shape[0] // bs * bs
    q, s = _pack(x[:n].reshape(-1, bs, *x.shape[1:]), codec)
    return torch.cat([(q.float() * s).reshape(n, *x.shape[1:]), x[n:]])


def _e4m3_64(y):
    """The nearest e4m3 value (ties to the even mantissa), by the format's spacing."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30)))
    step = torch.pow(torch.full_like(y, 2.0), torch.clamp_min(e, -6.0) - 3.0)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _held64(x, codec, bs):
    """_held from the definition: every f32 rounding step written out in 64 bits."""
    n = x.shape[0] // bs * bs
    v = x[:n].double().reshape(-1, bs, *x.shape[1:])
    a = torch.amax(v.abs(), dim=(1, 3))[:, None, :, None]
    top = _TOP[codec]
    zero = a < 2.0 ** -100
    a1 = torch.where(zero, 1.0, a)
    inv = (top / a1).float().double()
    sc = torch.where(zero, 0.0, (a1 / top).float().double())
    y = (v * inv).float().double()
    y = torch.round(y) if codec == "int8" else _e4m3_64(y)
    return torch.cat([(y * sc).reshape(n, *x.shape[1:]), x[n:].double()])


def _attend(q, k, v, first, scale):
    """Rows q [n, heads, hd] at positions first.. over k, v [t, kv_heads, hd], causal."""
    n, h, hd = q.shape
    kh = k.shape[1]
    qs = (q * scale).reshape(n, kh, h // kh, hd).permute(1, 2, 0, 3).reshape(kh, -1, hd).contiguous()
    s = torch.bmm(qs, k.permute(1, 2, 0).contiguous()).reshape(kh, h // kh, n, -1)
    hidden = torch.arange(k.shape[0], device=DEV)[None] > torch.arange(n, device=DEV)[:, None] + first
    s = torch.where(hidden, torch.full_like(s, -math.inf), s)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.bmm(p.reshape(kh, -1, k.shape[0]), v.permute(1, 0, 2).contiguous())
    o = o.reshape(kh, h // kh, n, hd) / p.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(n, h * hd)


# ---- rows of a cache: a shared run of rows, every sequence starting elsewhere in it

def _base_rows(g, c, layers, t):
    """K and V rows [layers, 2, t, kv_heads, hd]: unit scale with a few large channels,
    as keys have, and a size that drifts along the sequence."""
    w = (c["kv_heads"], c["hd"])
    x = _randn(g, layers, 2, t, *w)
    x *= 1.0 + 5.0 * (torch.rand(layers, 2, 1, *w, generator=g, device=DEV) > 0.97)
    return x * torch.exp(0.4 * torch.sin(torch.arange(t, device=DEV) / 37.0))[:, None, None]


def _rows(base, layer, side, s, first, n):
    t = base.shape[2]
    at = (torch.arange(first, first + n, device=DEV) + 13 * s) % t
    return base[layer, side][at]


def _new_cache(c, layers, seqs, max_time, pages, max_rows):
    from vokra_amd import hip
    codec = {"int8": hip.KvCodec.INT8, "e4m3": hip.KvCodec.E4M3}[c["codec"]]
    return _ctx().block_kv_cache(layers, c["kv_heads"], c["hd"], seqs, max_time, c["bs"], pages, max_rows, codec)


def _fill(kv, c, base, layers, seqs, starts, counts):
    """The rows starts..starts+counts of the sequences, as one step of the cache."""
    kv.step(seqs, starts, counts)
    for layer in range(layers):
        k, v = (torch.cat([_rows(base, layer, side, int(s), int(a), int(n)) for s, a, n in zip(seqs, starts, counts)])
                .contiguous() for side in (0, 1))
        torch.cuda.synchronize()
        kv.write_dev(layer, _Dev(k), _Dev(v))
        _ctx().synchronize()


def _fill_histories(kv, c, base, layers, lens, chunk):
    """Every sequence's first lens[s] rows, the sequences advancing together chunk by chunk."""
    done = np.zeros(len(lens), np.int64)
    while True:
        seqs = np.flatnonzero(done < lens)
        if not seqs.size:
            return
        counts = np.minimum(lens[seqs] - done[seqs], chunk)
        _fill(kv, c, base, layers, seqs, done[seqs], counts)
        done[seqs] += counts


def _cache_chunk(lens):
    return max(64, min(4096, 32768 // len(lens)))


# ---- family "attend": attention of a step's rows over the cache, every layer in turn

def _attend_shape(c, seed):
    order = np.random.default_rng(int(seed)).permutation(c["seqs"])
    lens = _spread(c["len_lo"], c["len_hi"], c["seqs"])  # rows held after the step
    counts = np.roll(_spread(c["count_lo"], c["count_hi"], c["seqs"]), c["seqs"] // 2)
    return lens[order], np.minimum(counts, lens)[order]


def _attend_inputs(c, seed):
    lens, counts = _attend_shape(c, seed)
    g = _gen(seed)
    base = _base_rows(g, c, c["layers"], int(lens.max()) + 64)
    q = _randn(g, c["layers"], int(counts.sum()), c["heads"] * c["hd"])
    return lens, counts, base, q


def _attend_prepare(c, seed):
    lens, counts, base, q = _attend_inputs(c, seed)
    layers, bs = c["layers"], c["bs"]
    if own:
        chunk = _cache_chunk(lens)
        kv = _new_cache(c, layers, c["seqs"], int(lens.max()), int((lens // bs).sum()) + 1,
                        max(int(counts.sum()), chunk * c["seqs"]))
        _fill_histories(kv, c, base, layers, lens - counts, chunk)
        _fill(kv, c, base, layers, np.arange(c["seqs"]), lens - counts, counts)
        o = [_Dev(torch.zeros_like(q[i])) for i in range(layers)]
        torch.cuda.synchronize()
        return {"kv": kv, "q": [_Dev(q[i]) for i in range(layers)], "o": o}
    packed = []
    for layer in range(layers):
        per = []
        for s in range(c["seqs"]):
            n = int(lens[s]) // bs * bs
            sides = []
            for side in (0, 1):
                x = _rows(base, layer, side, s, 0, int(lens[s]))
                sides.append((*_pack(x[:n].reshape(-1, bs, *x.shape[1:]), c["codec"]), x[n:].clone()))
            per.append(sides)
        packed.append(per)
    return {"packed": packed, "q": q, "lens": lens, "counts": counts}


def _unpack(side):
    q, s, rest = side
    return torch.cat([(q.float() * s).reshape(-1, *rest.shape[1:]), rest])


def _attend_run(c, s):
    if own:
        for layer in range(c["layers"]):
            s["kv"].attn_dev(layer, c["heads"], s["q"][layer], c["hd"] ** -0.5, s["o"][layer])
        return [o.t for o in s["o"]]
    out = []
    at = np.concatenate([[0], np.cumsum(s["counts"])])
    for layer in range(c["layers"]):
        rows = []
        for i in range(c["seqs"]):
            q = s["q"][layer, int(at[i]):int(at[i + 1])].reshape(-1, c["heads"], c["hd"])
            k, v = (_unpack(x) for x in s["packed"][layer][i])
            rows.append(_attend(q, k, v, int(s["lens"][i] - s["counts"][i]), c["hd"] ** -0.5))
        out.append(torch.cat(rows))
    return out


def _attend64(q, k, v, first, scale):
    """The definition in 64 bits, one kv head at a time: [rows, heads, hd] in, [rows, heads * hd] out."""
    n, h, hd = q.shape
    r = h // k.shape[1]
    out = torch.empty(n, h, hd, dtype=torch.float64, device=DEV)
    j = torch.arange(k.shape[0], device=DEV)
    for a in range(0, n, 128):
        b = min(n, a + 128)
        seen = j[None, :] <= (first + torch.arange(a, b, device=DEV))[:, None]
        for m in range(h):
            s = q[a:b, m].double() @ k[:, m // r].T.contiguous() * scale
            out[a:b, m] = torch.softmax(s.masked_fill(~seen, -math.inf), -1) @ v[:, m // r].contiguous()
    return out.reshape(n, h * hd)


def _attend_exact(c, seed):
    if _attend_work(c)["flops"] > 2e11:
        return None
    lens, counts, base, q = _attend_inputs(c, seed)
    at = np.concatenate([[0], np.cumsum(counts)])
    out = []
    for layer in range(c["layers"]):
        rows = []
        for i in range(c["seqs"]):
            k, v = (_held64(_rows(base, layer, side, i, 0, int(lens[i])), c["codec"], c["bs"]) for side in (0, 1))
            x = q[layer, int(at[i]):int(at[i + 1])].reshape(-1, c["heads"], c["hd"])
            rows.append(_attend64(x, k, v, int(lens[i] - counts[i]), c["hd"] ** -0.5))
        out.append(torch.cat(rows))
    return out


def _cache_bytes(c, lens):
    """K and V of one layer as the cache holds them."""
    w, bs = c["kv_heads"] * c["hd"], c["bs"]
    full = int((lens // bs).sum())
    return 2 * (full * (bs * w + 4 * c["kv_heads"]) + 4 * w * int((lens % bs).sum()))


def _attend_work(c):
    lens, counts = _attend_shape(c, 0)
    pairs = int((counts * lens - counts * (counts - 1) // 2).sum())
    return {"bytes": c["layers"] * (_cache_bytes(c, lens) + 8 * int(counts.sum()) * c["heads"] * c["hd"]),
            "flops": 4 * c["layers"] * c["heads"] * c["hd"] * pairs}


# ---- family "write": a step's rows into the cache of every layer, and what the cache then holds for them

def _write_prepare(c, seed):
    lens, counts = _attend_shape(c, seed)
    g = _gen(seed)
    base = _base_rows(g, c, c["layers"], int(lens.max()) + 64)
    starts = lens - counts
    new = [[torch.cat([_rows(base, layer, side, i, int(starts[i]), int(counts[i])) for i in range(c["seqs"])])
            .contiguous() for side in (0, 1)] for layer in range(c["layers"])]
    row_seq = np.repeat(np.arange(c["seqs"]), counts)
    row_time = np.concatenate([np.arange(a, a + n) for a, n in zip(starts, counts)])
    st = {"new": new, "starts": starts, "counts": counts, "lens": lens}
    if not own:
        st["before"] = [[[_rows(base, layer, side, i, int(starts[i]) // c["bs"] * c["bs"],
                                int(starts[i]) % c["bs"]) for i in range(c["seqs"])] for side in (0, 1)]
                        for layer in range(c["layers"])]
        return st
    chunk = _cache_chunk(lens)
    kv = _new_cache(c, c["layers"], c["seqs"], int(lens.max()), int((lens // c["bs"]).sum()) + c["seqs"],
                    max(int(counts.sum()), chunk * c["seqs"]))
    _fill_histories(kv, c, base, c["layers"], starts, chunk)
    st.update(kv=kv, seqs=_i32(np.arange(c["seqs"])), d_starts=_i32(starts), d_counts=_i32(counts),
              row_seq=_i32(row_seq), row_time=_i32(row_time), rows=[[_Dev(x) for x in p] for p in new],
              out=[[_Dev(torch.zeros_like(x)) for x in p] for p in new])
    torch.cuda.synchronize()
    return st


def _write_run(c, s):
    n = int(s["counts"].sum())
    if own:
        # a step may be taken back and repeated: its rows start where they started before
        if c["whole"]:  # prompts from their first row
            s["kv"].free_dev(c["seqs"], s["seqs"])
        s["kv"].step_dev(c["seqs"], n, int(s["counts"].max()), int(s["lens"].max()), s["seqs"], s["d_starts"],
                         s["d_counts"])
        for layer in range(c["layers"]):
            s["kv"].write_dev(layer, *s["rows"][layer])
        for layer in range(c["layers"]):
            s["kv"].read_dev(layer, n, s["row_seq"], s["row_time"], *s["out"][layer])
        return [[x.t for x in p] for p in s["out"]]
    at = np.concatenate([[0], np.cumsum(s["counts"])])
    out = []
    for layer in range(c["layers"]):
        sides = []
        for side in (0, 1):
            rows = []
            for i in range(c["seqs"]):
                old = s["before"][layer][side][i]
                x = torch.cat([old, s["new"][layer][side][int(at[i]):int(at[i + 1])]])
                rows.append(_held(x, c["codec"], c["bs"])[old.shape[0]:])
            sides.append(torch.cat(rows))
        out.append(sides)
    return out


def _write_exact(c, seed):
    lens, counts = _attend_shape(c, seed)
    base = _base_rows(_gen(seed), c, c["layers"], int(lens.max()) + 64)
    out = []
    for layer in range(c["layers"]):
        sides = []
        for side in (0, 1):
            rows = []
            for i in range(c["seqs"]):
                first = int(lens[i] - counts[i])
                a = first // c["bs"] * c["bs"]
                rows.append(_held64(_rows(base, layer, side, i, a, int(lens[i]) - a), c["codec"], c["bs"])[first - a:])
            sides.append(torch.cat(rows))
        out.append(sides)
    return out


def _write_work(c):
    lens, counts = _attend_shape(c, 0)
    n, w = int(counts.sum()), c["kv_heads"] * c["hd"]
    held = 2 * n * w  # 8-bit values written and read back
    return {"bytes": c["layers"] * (2 * n * w * 4 + 2 * held + 2 * n * w * 4), "flops": 0}


# ---- family "beam": a step of several candidates per prompt: the last candidates' pages are freed, new ones
# forked from the prompts' sequences, one row each written and attended, in every layer

def _beam_inputs(c, seed):
    rng = np.random.default_rng(int(seed))
    lens = rng.permutation(_spread(c["len_lo"], c["len_hi"], c["seqs"]))
    src = rng.integers(0, c["seqs"], c["seqs"] * c["beams"])  # a candidate's parent
    g = _gen(seed)
    base = _base_rows(g, c, c["layers"], int(lens.max()) + 64)
    n = src.size
    new = _randn(g, c["layers"], 2, n, c["kv_heads"], c["hd"])
    q = _randn(g, c["layers"], n, c["heads"] * c["hd"])
    return lens, src, base, new, q


def _beam_prepare(c, seed):
    lens, src, base, new, q = _beam_inputs(c, seed)
    layers, bs, n = c["layers"], c["bs"], src.size
    if not own:
        rows = [[[_rows(base, layer, side, s, 0, int(lens[s])) for s in range(c["seqs"])] for side in (0, 1)]
                for layer in range(layers)]
        packed = [[[(*_pack(x[:x.shape[0] // bs * bs].reshape(-1, bs, *x.shape[1:]), c["codec"]),
                     x[x.shape[0] // bs * bs:].clone()) for x in sides] for sides in per] for per in rows]
        return {"packed": packed, "src": src, "lens": lens, "new": new, "q": q}
    chunk = _cache_chunk(lens)
    kv = _new_cache(c, layers, c["seqs"] + n, int(lens.max()) + 1, int((lens // bs).sum()) + n + 1,
                    max(n, chunk * c["seqs"]))
    _fill_histories(kv, c, base, layers, lens, chunk)
    st = {"kv": kv, "n": n, "src": _i32(src), "dst": _i32(c["seqs"] + np.arange(n)), "starts": _i32(lens[src]),
          "ones": _i32(np.ones(n)), "max": int(lens.max()) + 1, "new": [[_Dev(x.contiguous()) for x in p] for p in new],
          "q": [_Dev(x) for x in q], "o": [_Dev(torch.zeros_like(x)) for x in q]}
    torch.cuda.synchronize()
    return st


def _beam_run(c, s):
    if own:
        kv, n = s["kv"], s["n"]
        kv.free_dev(n, s["dst"])
        kv.fork_dev(n, s["src"], s["dst"])
        kv.step_dev(n, n, 1, s["max"], s["dst"], s["starts"], s["ones"])
        for layer in range(c["layers"]):
            kv.write_dev(layer, *s["new"][layer])
            kv.attn_dev(layer, c["heads"], s["q"][layer], c["hd"] ** -0.5, s["o"][layer])
        return [o.t for o in s["o"]]
    out = []
    for layer in range(c["layers"]):
        rows = []
        for i, p in enumerate(s["src"]):
            sides = []
            for side in (0, 1):
                q, sc, rest = s["packed"][layer][side][p]
                rest = torch.cat([rest, s["new"][layer, side, i:i + 1]])
                sides.append(torch.cat([(q.float() * sc).reshape(-1, *rest.shape[1:]),
                                        _held(rest, c["codec"], c["bs"])]))
            q = s["q"][layer, i].reshape(1, c["heads"], c["hd"])
            rows.append(_attend(q, *sides, int(s["lens"][p]), c["hd"] ** -0.5))
        out.append(torch.cat(rows))
    return out


def _beam_exact(c, seed):
    lens, src, base, new, q = _beam_inputs(c, seed)
    out = []
    for layer in range(c["layers"]):
        rows = []
        for i, p in enumerate(src):
            k, v = (_held64(torch.cat([_rows(base, layer, side, int(p), 0, int(lens[p])), new[layer, side, i:i + 1]]),
                            c["codec"], c["bs"]) for side in (0, 1))
            rows.append(_attend64(q[layer, i].reshape(1, c["heads"], c["hd"]), k, v, int(lens[p]), c["hd"] ** -0.5))
        out.append(torch.cat(rows))
    return out


def _beam_work(c):
    lens = _spread(c["len_lo"], c["len_hi"], c["seqs"])
    n, w = c["seqs"] * c["beams"], c["kv_heads"] * c["hd"]
    rows = n * (2 * w * 4 + 2 * c["heads"] * c["hd"] * 4)
    # the prompts' pages are shared: read once; the open block's rows go to every candidate
    mean_open = int((lens % c["bs"]).sum()) / c["seqs"]
    forked = 2 * 2 * 4 * w * mean_open * n
    return {"bytes": c["layers"] * (_cache_bytes(c, lens) + rows + forked),
            "flops": 4 * c["layers"] * c["heads"] * c["hd"] * c["beams"] * int((lens + 1).sum())}


# ---- family "handover": prompts' pages copied from one cache into another, half of them given up again, the rest
# compacted, and read (as when finished prompts move to the cache that serves them)

def _handover_inputs(c, seed):
    rng = np.random.default_rng(int(seed))
    order = rng.permutation(c["seqs"])
    lens = _spread(c["len_lo"], c["len_hi"], c["seqs"])[order]
    kept = np.flatnonzero(order % 2 == 0)  # every second one by length
    base = _base_rows(_gen(seed), c, c["layers"], int(lens.max()) + 64)
    return lens, rng.permutation(c["seqs"]), kept, base


def _handover_prepare(c, seed):
    lens, dst, kept, base = _handover_inputs(c, seed)
    layers, bs = c["layers"], c["bs"]
    if not own:
        packed = [[[(*_pack(x[:x.shape[0] // bs * bs].reshape(-1, bs, *x.shape[1:]), c["codec"]),
                     x[x.shape[0] // bs * bs:].clone())
                    for x in (_rows(base, layer, side, int(s), 0, int(lens[s])) for s in kept)] for side in (0, 1)]
                  for layer in range(layers)]
        return {"packed": packed}
    chunk = _cache_chunk(lens)
    pages = int((lens // bs).sum()) + 1
    a = _new_cache(c, layers, c["seqs"], int(lens.max()), pages, chunk * c["seqs"])
    b = _new_cache(c, layers, c["seqs"], int(lens.max()), pages, 1)
    _fill_histories(a, c, base, layers, lens, chunk)
    n = int(lens[kept].sum())
    w = c["kv_heads"], c["hd"]
    st = {"a": a, "b": b, "src": _i32(np.arange(c["seqs"])), "dst": _i32(dst), "gone": _i32(np.delete(dst, kept)),
          "rows": n, "row_seq": _i32(np.repeat(dst[kept], lens[kept])),
          "row_time": _i32(np.concatenate([np.arange(lens[s]) for s in kept])),
          "out": [[_Dev(torch.zeros(n, *w, device=DEV)) for _ in (0, 1)] for _ in range(layers)]}
    torch.cuda.synchronize()
    return st


def _handover_run(c, s):
    if own:
        b = s["b"]
        b.free_dev(c["seqs"], s["src"])
        b.copy_from_dev(s["a"], c["seqs"], s["src"], s["dst"])
        b.free_dev(s["gone"].t.numel(), s["gone"])
        b.compact()
        for layer in range(c["layers"]):
            b.read_dev(layer, s["rows"], s["row_seq"], s["row_time"], *s["out"][layer])
        return [[x.t for x in p] for p in s["out"]]
    out = []
    for per in s["packed"]:
        sides = []
        for side in per:
            moved = [(q.clone(), sc.clone(), rest.clone()) for q, sc, rest in side]
            sides.append(torch.cat([_unpack(x) for x in moved]))
        out.append(sides)
    return out


def _handover_exact(c, seed):
    lens, _, kept, base = _handover_inputs(c, seed)
    return [[torch.cat([_held64(_rows(base, layer, side, int(s), 0, int(lens[s])), c["codec"], c["bs"]) for s in kept])
             for side in (0, 1)] for layer in range(c["layers"])]


def _handover_work(c):
    lens = _spread(c["len_lo"], c["len_hi"], c["seqs"])
    kept = lens[::2]
    w = c["kv_heads"] * c["hd"]
    # every page read and written by the copy; the kept ones read; their rows written
    return {"bytes": c["layers"] * (2 * _cache_bytes(c, lens) + _cache_bytes(c, kept) + 8 * w * int(kept.sum())),
            "flops": 0}


# ---- family "rope": q and k rows of a step turned to their positions

def _rope_freqs(c):
    """Radians per position of each pair, and the factor on the turned values (64 bits)."""
    r, base, f = c["rot"], c["base"], c["factor"]
    j = np.arange(r // 2, dtype=np.float64)
    if c["scaling"] == "ntk":
        return (base * f ** (r / (r - 2))) ** (-2 * j / r), 1.0
    th = base ** (-2 * j / r)
    if c["scaling"] == "linear":
        return th / f, 1.0
    if c["scaling"] == "yarn":
        def at(turns):  # the pair that makes `turns` turns over the trained context
            return r * math.log(c["orig"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        ramp = np.clip((j - lo) / max(hi - lo, 0.001), 0, 1)
        return th / f * ramp + th * (1 - ramp), 0.1 * math.log(f) + 1.0
    if c["scaling"] == "bands":
        turns = c["orig"] * th / (2 * math.pi)  # over the trained context; 1 .. 4 turns blend
        mix = np.clip((turns - 1.0) / 3.0, 0, 1)
        return th / f * (1 - mix) + th * mix, 1.0
    return th, 1.0


def _rope_inputs(c, seed):
    g = _gen(seed)
    rng = np.random.default_rng(int(seed))
    width = (c["heads"] + 2 * c["kv_heads"]) * c["hd"]  # q, k and v rows side by side, as one projection leaves them
    qkv = _randn(g, c["rows"], width)
    first = rng.integers(0, c["pos_hi"] - c["run"] + 2, -(-c["rows"] // c["run"]))
    pos = (first[:, None] + np.arange(c["run"])).reshape(-1)[:c["rows"]]
    return qkv, pos


def _rope_prepare(c, seed):
    qkv, pos = _rope_inputs(c, seed)
    th, mag = _rope_freqs(c)
    st = {"qkv": qkv, "pos": torch.as_tensor(pos, device=DEV, dtype=torch.int32)}
    if not own:
        st.update(th=torch.as_tensor(th, device=DEV), mag=mag)
        return st
    from vokra_amd import hip
    kind = {"none": hip.RopeScaling.NONE, "linear": hip.RopeScaling.LINEAR, "ntk": hip.RopeScaling.NTK,
            "yarn": hip.RopeScaling.YARN, "bands": hip.RopeScaling.BANDS}[c["scaling"]]
    layout = {"half": hip.RopeLayout.HALF, "pairs": hip.RopeLayout.INTERLEAVED}[c["layout"]]
    st.update(plan=_ctx().rope_plan(c["hd"], c["rot"], layout, c["base"], kind, c["factor"], c["orig"]),
              d_pos=_Dev(st["pos"]), q=_Dev(qkv), k=_Dev(qkv.reshape(-1)[c["heads"] * c["hd"]:]),
              qo=_Dev(torch.zeros(c["rows"], c["heads"] * c["hd"], device=DEV)),
              ko=_Dev(torch.zeros(c["rows"], c["kv_heads"] * c["hd"], device=DEV)))
    torch.cuda.synchronize()
    return st


def _rope_run(c, s):
    hd, rot, h = c["hd"], c["rot"], c["heads"] + c["kv_heads"]
    if own:
        width = s["qkv"].shape[1]
        s["plan"].apply_dev(c["rows"], s["d_pos"], c["heads"], s["q"], s["qo"], c["kv_heads"], s["k"], s["ko"],
                            q_stride=width, k_stride=width)
        return {"q": s["qo"].t, "k": s["ko"].t}
    ang = s["pos"].double()[:, None] * s["th"]
    cs, sn = ((f(ang) * s["mag"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = s["qkv"][:, :h * hd].reshape(-1, h, hd)
    y = x.clone()
    if c["layout"] == "half":
        a, b = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        a, b = slice(0, rot, 2), slice(1, rot, 2)
    y[..., a] = x[..., a] * cs - x[..., b] * sn
    y[..., b] = x[..., a] * sn + x[..., b] * cs
    y = y.reshape(-1, h * hd)
    return {"q": y[:, :c["heads"] * hd].contiguous(), "k": y[:, c["heads"] * hd:].contiguous()}


def _rope_exact(c, seed):
    qkv, pos = _rope_inputs(c, seed)
    th, mag = _rope_freqs(c)
    hd, rot = c["hd"], c["rot"]
    turn = torch.polar(torch.full((c["rows"], rot // 2), mag, dtype=torch.float64, device=DEV),
                       torch.as_tensor(pos[:, None] * th[None], device=DEV))[:, None]
    got = {}
    for name, lo, n in (("q", 0, c["heads"]), ("k", c["heads"] * hd, c["kv_heads"])):
        x = qkv[:, lo:lo + n * hd].double().reshape(-1, n, hd)
        head = x[..., :rot].reshape(-1, n, 2, rot // 2).transpose(-1, -2) if c["layout"] == "half" else \
            x[..., :rot].reshape(-1, n, rot // 2, 2)
        z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn)
        z = z.transpose(-1, -2).reshape(-1, n, rot) if c["layout"] == "half" else z.reshape(-1, n, rot)
        got[name] = torch.cat([z, x[..., rot:]], -1).reshape(-1, n * hd)
    return got


def _rope_work(c):
    n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["hd"]
    return {"bytes": 8 * n + 4 * c["rows"], "flops": 3 * n * c["rot"] // c["hd"]}


# ---- family "rules": logits through a step's penalties, biases and grammar masks, and the greedy choice

def _rules_inputs(c, seed):
    g = _gen(seed)
    rng = np.random.default_rng(int(seed))
    rows, vocab = c["rows"], c["vocab"]
    logits = _randn(g, rows, vocab) * 3.0
    lens = rng.permutation(_spread(c["hist_lo"], c["hist_hi"], rows))
    # words repeat: tokens come from a few hundred of the vocabulary, some of them often
    pool = rng.integers(0, vocab, 400)
    hist = pool[np.minimum(rng.geometric(0.02, int(lens.sum())) - 1, 399)]
    nb = np.full(rows, c["biases"])
    ids = rng.integers(0, vocab, int(nb.sum()))
    bias = rng.normal(0, 4, ids.size).astype(np.float32)
    pen = np.stack([rng.uniform(1.0, 1.4, rows), rng.uniform(0.0, 1.0, rows), rng.uniform(0.0, 0.5, rows)])
    words = -(-vocab // 32)
    mask = None
    if c["mask"]:
        mask = rng.integers(0, 1 << 32, (rows, words), dtype=np.uint64)
        for _ in range(3):  # a grammar leaves few tokens: a sixteenth of the bits, some rows none
            mask &= rng.integers(0, 1 << 32, (rows, words), dtype=np.uint64)
        mask[rng.random(rows) < 0.02] = 0
        mask = mask.astype(np.uint32)
    off = lambda n: np.concatenate([[0], np.cumsum(n)]).astype(np.int32)  # noqa: E731
    return {"logits": logits, "hist": hist, "hist_off": off(lens), "ids": ids, "bias": bias, "bias_off": off(nb),
            "pen": pen.astype(np.float32), "mask": mask}


def _rules_prepare(c, seed):
    x = _rules_inputs(c, seed)
    d = {k: torch.as_tensor(v, device=DEV) for k, v in x.items() if k not in ("mask", "logits")}
    d["logits"] = x["logits"]
    d["mask"] = None if x["mask"] is None else torch.as_tensor(x["mask"].view(np.int32), device=DEV)
    if not own:
        rows = torch.arange(c["rows"], device=DEV)
        d["hist_row"] = torch.repeat_interleave(rows, d["hist_off"].diff().long())
        d["bias_row"] = torch.repeat_interleave(rows, d["bias_off"].diff().long())
        return d
    from vokra_amd import hip
    keep = {k: _Dev(d[k].to(torch.int32).contiguous()) for k in ("hist", "hist_off", "ids", "bias_off")}
    keep.update(bias=_Dev(d["bias"]), pen=[_Dev(d["pen"][i].clone()) for i in range(3)],
                mask=None if d["mask"] is None else _Dev(d["mask"]))
    rules = hip.LogitsRules(n_hist=int(x["hist"].size), hist=keep["hist"], hist_offsets=keep["hist_off"],
                            repetition=keep["pen"][0], presence=keep["pen"][1], frequency=keep["pen"][2],
                            n_bias=int(x["ids"].size), bias_ids=keep["ids"], bias=keep["bias"],
                            bias_offsets=keep["bias_off"], mask=keep["mask"],
                            mask_stride=-(-c["vocab"] // 32) if c["mask"] else 0)
    st = {"rules": rules, "keep": keep, "logits": _Dev(d["logits"]), "out": _Dev(torch.zeros_like(d["logits"])),
          "next": _Dev(torch.zeros(c["rows"], dtype=torch.int32, device=DEV))}
    torch.cuda.synchronize()
    return st


def _rules_run(c, s):
    if own:
        _ctx().logits_rules_dev(c["rows"], c["vocab"], s["logits"], s["rules"], s["out"], s["next"])
        return {"logits": s["out"].t, "next": s["next"].t}
    rows, vocab = c["rows"], c["vocab"]
    x = s["logits"]
    count = torch.zeros(rows * vocab, device=DEV, dtype=torch.int32)
    at = s["hist_row"] * vocab + s["hist"].long()
    count.index_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    count = count.reshape(rows, vocab)
    rep, pres, freq = (s["pen"][i][:, None] for i in range(3))
    y = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep), x)
    y = torch.where(count > 0, y - (pres + freq * count.float()), y)
    slot = torch.full((rows * vocab,), -1, device=DEV, dtype=torch.int64)
    at = s["bias_row"] * vocab + s["ids"].long()
    slot.scatter_reduce_(0, at, torch.arange(at.numel(), device=DEV), "amax")  # an id given twice: the last counts
    slot = slot.reshape(rows, vocab)
    if at.numel():
        y = torch.where(slot >= 0, y + s["bias"][slot.clamp_min(0)], y)
    if s["mask"] is not None:
        bit = torch.arange(vocab, device=DEV)
        y = torch.where(((s["mask"][:, bit // 32] >> (bit % 32)) & 1) > 0, y, torch.full_like(y, -math.inf))
    top = y.amax(1, keepdim=True)
    idx = torch.where(y == top, torch.arange(vocab, device=DEV)[None], vocab).amin(1)
    nxt = torch.where(top[:, 0] > -math.inf, idx, torch.full_like(idx, -1))
    return {"logits": y, "next": nxt.to(torch.int32)}


def _rules_exact(c, seed):
    x = _rules_inputs(c, seed)
    y = x["logits"].double().cpu().numpy()
    nxt = np.empty(c["rows"], np.int32)
    for r in range(c["rows"]):
        h, n = np.unique(x["hist"][x["hist_off"][r]:x["hist_off"][r + 1]], return_counts=True)
        rep, pres, freq = (float(p[r]) for p in x["pen"])
        l = y[r, h]
        y[r, h] = np.where(l > 0, l / rep, l * rep) - (pres + freq * n)
        b = slice(x["bias_off"][r], x["bias_off"][r + 1])
        last = dict(zip(x["ids"][b].tolist(), x["bias"][b].tolist()))
        if last:
            y[r, list(last)] += np.array(list(last.values()))
        if x["mask"] is not None:
            bits = np.unpackbits(x["mask"][r].view(np.uint8), bitorder="little")[:c["vocab"]]
            y[r, bits == 0] = -np.inf
        nxt[r] = -1 if not np.any(y[r] > -np.inf) else int(np.argmax(y[r]))
    return {"logits": y, "next": nxt}


def _rules_work(c):
    lens = _spread(c["hist_lo"], c["hist_hi"], c["rows"])
    n = c["rows"] * c["vocab"]
    return {"bytes": 8 * n + (n // 8 if c["mask"] else 0) + 4 * int(lens.sum()) + 8 * c["rows"] * c["biases"],
            "flops": 4 * n}


# ---- the cases -----------------------------------------------------------------

_FAMILY = {"attend": (_attend_prepare, _attend_run, _attend_exact, _attend_work),
           "write": (_write_prepare, _write_run, _write_exact, _write_work),
           "beam": (_beam_prepare, _beam_run, _beam_exact, _beam_work),
           "handover": (_handover_prepare, _handover_run, _handover_exact, _handover_work),
           "rope": (_rope_prepare, _rope_run, _rope_exact, _rope_work),
           "rules": (_rules_prepare, _rules_run, _rules_exact, _rules_work)}


def _case(family, name=None, **kw):
    c = {"family": family, **kw}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the first tokens of a few streams of a speech decoder: the call's latency
        _case("attend", "attend_first_tokens", codec="int8", bs=16, hd=64, heads=20, kv_heads=20, layers=4, seqs=4,
              len_lo=1, len_hi=50, count_lo=1, count_hi=1),
        # a decode step of a speech LLM's streams over mixed contexts
        _case("attend", "attend_streams", codec="int8", bs=16, hd=128, heads=16, kv_heads=2, layers=6, seqs=32,
              len_lo=512, len_hi=4096, count_lo=1, count_hi=1),
        # few long documents in 8-bit floats, several drafted tokens checked at once
        _case("attend", "attend_long_drafts", codec="e4m3", bs=64, hd=128, heads=32, kv_heads=8, layers=1, seqs=6,
              len_lo=9001, len_hi=65001, count_lo=1, count_hi=4),
        # prompts of a batch taken in chunks behind histories of their own
        _case("attend", "attend_chunks", codec="int8", bs=32, hd=128, heads=16, kv_heads=2, layers=1, seqs=6,
              len_lo=700, len_hi=4500, count_lo=450, count_hi=1030),
        # one decode step's rows of 64 streams, 8 layers
        _case("write", "write_token", codec="int8", bs=16, hd=64, heads=20, kv_heads=20, layers=8, seqs=64,
              len_lo=1, len_hi=448, count_lo=1, count_hi=1, whole=False),
        # a batch of whole prompts
        _case("write", "write_prompts", codec="e4m3", bs=32, hd=128, heads=16, kv_heads=8, layers=4, seqs=8,
              len_lo=333, len_hi=4097, count_lo=4097, count_hi=4097, whole=True),
        # beam search: four candidates of each of eight prompts
        _case("beam", "beam_step", codec="int8", bs=16, hd=128, heads=16, kv_heads=2, layers=6, seqs=8,
              beams=4, len_lo=100, len_hi=2000),
        # prompts moved to the serving cache
        _case("handover", "handover_prompts", codec="int8", bs=16, hd=128, heads=16, kv_heads=4, layers=8, seqs=16,
              len_lo=200, len_hi=3000),
        # a decode step's q and k
        _case("rope", "rope_step", layout="half", hd=128, rot=128, heads=16, kv_heads=2, rows=32, run=1,
              pos_hi=4096, base=10000.0, scaling="none", factor=1.0, orig=4096),
        # long prompts, half of each head turned in pairs, scaled to eight times the trained context
        _case("rope", "rope_prompts", layout="pairs", hd=128, rot=64, heads=32, kv_heads=8, rows=8191, run=2730,
              pos_hi=131072, base=500000.0, scaling="yarn", factor=8.0, orig=16384),
        # the constrained streams of a speech LLM
        _case("rules", "rules_streams", rows=32, vocab=32000, hist_lo=0, hist_hi=4096, biases=20, mask=True),
        # a large batch over a large vocabulary with penalties alone
        _case("rules", "rules_large", rows=192, vocab=128259, hist_lo=1, hist_hi=2048, biases=300, mask=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(["attend", "attend", "attend", "write", "beam", "handover", "rope", "rules"])
    cache = dict(codec=rng.choice(["int8", "e4m3"]), bs=rng.choice([16, 32, 64]), hd=rng.choice([64, 128]))
    kv_heads = rng.choice([1, 2, 3, 4, 8, 20])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8] if kv_heads < 20 else [1])
    w = kv_heads * cache["hd"]
    layers = rng.randint(1, 3)
    if family == "attend":
        how = rng.choice(["token", "token", "draft", "chunk"])
        seqs = _log(rng, 1, 96) if how == "token" else _log(rng, 1, 12)
        count_lo, count_hi = 1, 1
        if how == "chunk":
            count_hi = _log(rng, 17, 1500)
            count_lo = rng.randint(1, count_hi)
            most = 8e10 / (4 * layers * heads * cache["hd"] * seqs * count_hi)
        else:
            count_hi = rng.randint(2, 16) if how == "draft" else 1
            most = (3e7 if how == "draft" else 7e7) / (seqs * w)
        hi = _log(rng, 8, max(8, min(65000, int(most))))
        return _case("attend", **cache, heads=heads, kv_heads=kv_heads, layers=layers, seqs=seqs,
                     len_lo=rng.randint(1, hi), len_hi=hi, count_lo=count_lo, count_hi=count_hi)
    if family == "write":
        whole = rng.random() < 0.5
        seqs = _log(rng, 1, 12) if whole else _log(rng, 1, 200)
        hi = _log(rng, 5, max(5, min(4000 if whole else 600, int(4e7 / (seqs * w * layers)))))
        return _case("write", **cache, heads=heads, kv_heads=kv_heads, layers=layers, seqs=seqs,
                     len_lo=rng.randint(1, hi), len_hi=hi, count_lo=hi if whole else 1,
                     count_hi=hi if whole else rng.randint(1, 16), whole=whole)
    if family == "beam":
        hi = _log(rng, 3, 2000)
        return _case("beam", **cache, heads=heads, kv_heads=kv_heads, layers=layers, seqs=_log(rng, 1, 8),
                     beams=rng.randint(1, 6), len_lo=rng.randint(1, hi), len_hi=hi)
    if family == "handover":
        seqs = _log(rng, 2, 16)
        hi = _log(rng, 3, min(2500, int(1e8 / (seqs * w * layers))))
        return _case("handover", **cache, heads=heads, kv_heads=kv_heads, layers=layers, seqs=seqs,
                     len_lo=rng.randint(1, hi), len_hi=hi)
    if family == "rope":
        hd = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([hd, hd // 2, hd // 4, rng.randint(2, hd // 2) * 2])
        rows = _log(rng, 1, 8000)
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        return _case("rope", layout=rng.choice(["half", "pairs"]), hd=hd, rot=max(4, rot // 2 * 2), heads=heads,
                     kv_heads=min(kv_heads, 8), rows=min(rows, int(3e7 / ((heads + kv_heads) * hd))),
                     run=rng.choice([1, 7, 500]), pos_hi=_log(rng, 600, 1000000), base=rng.choice([10000.0, 500000.0]),
                     scaling=scaling, factor=1.0 if scaling == "none" else rng.uniform(1.5, 32.0),
                     orig=_log(rng, 2048, 32768))
    vocab = _log(rng, 1000, 150000)
    hi = _log(rng, 1, 8000)
    return _case("rules", rows=min(_log(rng, 1, 256), int(2.4e7 / vocab)), vocab=vocab, hist_lo=rng.randint(0, hi),
                 hist_hi=hi, biases=rng.choice([0, 1, 40, 300]), mask=rng.random() < 0.6)


def prepare(case, seed):
    c = dict(case)
    state = _FAMILY[c["family"]][0](c, seed)
    state["case"] = c
    return state


def run(state):
    c = state["case"]
    return _FAMILY[c["family"]][1](c, state)


def exact(case, seed):
    c = dict(case)
    return _FAMILY[c["family"]][2](c, seed)


def work(case):
    c = dict(case)
    return _FAMILY[c["family"]][3](c)
