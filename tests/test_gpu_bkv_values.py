"""GPU parity of the block-scaled cache's attention at values that few caches hold:
zero blocks beside small ones, both ends of f32, blocks that are not finite at the
causal edge. The restatement and its bound are those of bkv_model."""
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


def attend(ctx, p, t, count, heads, far, q=None):
    """The last `count` of sequence 0's t rows as a step (the rows before it are
    there): (out, restated out, bound). far: a step sized for long sequences,
    which takes 17 to 96 columns in tiles of 32 and more in tiles of 128."""
    hd = p.ref.hd
    q = p.g.standard_normal((count, heads * hd)).astype(np.float32) if q is None else q
    up = lambda a: hip.DeviceBuffer.from_array(ctx, a)  # noqa: E731
    ids = [_Ids(ctx, [x]) for x in (0, t - count, count)]
    p.dev.step_dev(1, count, count, 1 << 24 if far else t, *ids)
    assert p.ref.step([0], [t - count], [count]) == (bm.OK, 1) and p.dev.status() == 1
    k, v = p.tail
    d = [up(x) for x in (k, v, q)]
    out = up(np.full(q.shape, 7.5, np.float32))
    p.dev.write_dev(0, d[0], d[1])
    p.ref.write(0, k, v)
    p.dev.attn_dev(0, heads, d[2], hd ** -0.5, out)
    ctx.synchronize()
    with np.errstate(invalid="ignore"):
        want, tol = p.ref.attn(0, q, heads, np.float32(hd ** -0.5))
    return out.download(np.float32, q.size).reshape(q.shape).astype(np.float64), want, tol


def filled(ctx, codec, hd, t, count, size, far, k_size=0.3, seed=0):
    """A cache of one sequence and one head: t - count rows written, the others in
    p.tail; row j's values are of magnitude size[j]."""
    bs = 16
    p = Pair(ctx, 1, 1, hd, 1, 1 << 20 if far else t, bs, t // bs + 1, t, codec, seed)
    k = (p.g.standard_normal((t, hd)) * k_size).astype(np.float32)
    v = (p.g.uniform(-1, 1, (t, hd)) * size[:, None]).astype(np.float32)
    first = t - count
    p.ref.step([0], [0], [first])
    p.dev.step([0], [0], [first])
    p.dev.write(0, k[:first], v[:first])
    p.ref.write(0, k[:first], v[:first])
    p.tail = k[first:], v[first:]
    return p


@pytest.mark.parametrize("codec,hd,count,heads,far", [(0, 128, 2, 4, False), (1, 64, 12, 4, True), (0, 64, 12, 12, True)])
def test_nan_block_reaches_rows_that_hardly_weigh_it(ctx, codec, hd, count, heads, far):
    """A key's weight may be 2^-600: its block reads as NaN all the same, at the causal
    edge (the block shares its 32 keys with hidden ones) as anywhere."""
    for behind in (0, 8, 16, 64):  # rows between the block and the step's
        print("[case] bkv nan of no weight", codec, hd, count, heads, far, behind, flush=True)
        t = 16 + behind + count
        p = filled(ctx, codec, hd, t, count, np.ones(t), far)
        k, v = (np.concatenate([x[0, :t - count].reshape(-1, hd), y])
                for x, y in zip(p.ref.rows[0][0][:, None], p.tail))
        k[:] = 0
        k[:16] = -40
        v[5, 3] = np.nan
        p.both("free", [0])
        first = t - count
        p.ref.step([0], [0], [first])
        p.dev.step([0], [0], [first])
        p.dev.write(0, k[:first], v[:first])
        p.ref.write(0, k[:first], v[:first])
        p.tail = k[first:], v[first:]
        got, want, _ = attend(ctx, p, t, count, heads, far, np.ones((count, heads * hd), np.float32))
        assert np.all(np.isnan(want)) and np.all(np.isnan(got))


@pytest.mark.parametrize("count,heads,far", [(3, 4, False), (20, 4, True), (20, 8, True)])
def test_nan_blocks_of_either_side_stay_hidden_from_earlier_rows(ctx, count, heads, far):
    """Rows before a block with a NaN in K or V do not see it, rows in or behind it do."""
    for side in (0, 1):
        for t, at in ((32, 30), (41, 40), (48, 45), (605, 602), (41, 41 - count), (605, 605 - count)):
            print("[case] bkv nan hidden", count, heads, far, side, t, at, flush=True)
            p = filled(ctx, 0, 64, t, count, np.ones(t), far, seed=t)
            k, v = p.tail
            (k, v)[side][at - t, 5] = np.nan
            got, want, tol = attend(ctx, p, t, count, heads, far)
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any()
            err = np.abs(got - want) / tol
            assert not np.any(err > 1), f"{np.nanmax(err)} of the bound"


# (magnitudes of the blocks in turn, of the open block's rows)
SIZES = [([0, 1e-6], 1e-6), ([0, 1e-8, 1e-8], 1e-8), ([1e-10, 0], 0), ([1e-8], 0), ([1e-12, 0, 0], 1e-12),
         ([0], 1e-12), ([0], 1e-33), ([1e20, 1e-20], 1e-20), ([1e-20], 1e20), ([1e-28, 0, 1e-28], 1e-33),
         ([3.4e38, 1e-30, 0], 1.0), ([1.0, 0], 3.4e38), ([0], 0)]


@pytest.mark.parametrize("count,t,far", [(2, 605, False), (12, 605, True), (24, 2100, False), (40, 605, True)])
@pytest.mark.parametrize("codec,hd", [(0, 128), (1, 64)])
def test_attention_of_values_far_apart(ctx, codec, hd, count, t, far):
    """Blocks of zeros have no part in how far small blocks' weights are rounded, and a
    key counts in the sum of weights whatever its values are: one and several key
    ranges, tiles of 16, 32 and 128 columns."""
    for n, (sizes, rest) in enumerate(SIZES):
        print("[case] bkv far apart", codec, hd, count, t, far, sizes, rest, flush=True)
        size = np.repeat(np.resize(sizes, t // 16 + 1), 16)[:t].astype(np.float64)
        size[t // 16 * 16:] = rest
        p = filled(ctx, codec, hd, t, count, size, far, seed=n)
        got, want, tol = attend(ctx, p, t, count, 4, far)
        assert np.all(np.isfinite(want))
        err = np.abs(got - want) / tol
        assert np.all(err <= 1), f"{err.max()} of the bound"


def test_attention_under_a_negative_scale(ctx):
    """A scale below zero turns the order of the scores round; zero weighs all alike."""
    for scale in (-0.125, 0.0):
        print("[case] bkv scale", scale, flush=True)
        p = Pair(ctx, 1, 2, 64, 2, 300, 16, 40, 600)
        p.step([0, 1], [0, 0], [290, 45])
        p.check_attn(0, 335, 4, scale)
        p.step([0, 1], [290, 45], [1, 3])
        p.check_attn(0, 4, 4, scale)


def test_one_buffer_for_q_and_the_output_is_refused(ctx):
    print("[case] bkv attn one buffer", flush=True)
    kv = ctx.block_kv_cache(1, 2, 64, 3, 100, 16, 10, 64)
    kv.step([0, 1], [0, 0], [3, 2])
    q, out = (hip.DeviceBuffer.from_array(ctx, np.zeros(5 * 256, np.float32)) for _ in (0, 1))
    with pytest.raises(hip.InvalidArgument):
        kv.attn_dev(0, 4, q, 0.125, q)
    kv.attn_dev(0, 4, q, 0.125, out)
    ctx.synchronize()


@pytest.mark.parametrize("first,count,heads,far", [(250, 22, 2, False), (250, 5, 2, False), (2040, 48, 2, False),
                                                   (505, 30, 4, False), (250, 60, 4, True), (250, 300, 2, True)])
@pytest.mark.parametrize("codec,hd", [(0, 64), (1, 128)])
def test_key_ranges_hidden_from_a_tiles_first_rows(ctx, codec, hd, first, count, heads, far):
    """The last key range of a tile begins behind its first rows, which have no key in it."""
    print("[case] bkv hidden range", codec, hd, first, count, heads, far, flush=True)
    t = first + count
    p = filled(ctx, codec, hd, t, count, np.ones(t), far, seed=t)
    got, want, tol = attend(ctx, p, t, count, heads, far)
    err = np.abs(got - want) / tol
    assert np.all(err <= 1), f"{np.nanmax(err)} of the bound"
