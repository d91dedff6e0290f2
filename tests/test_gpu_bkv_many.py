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
