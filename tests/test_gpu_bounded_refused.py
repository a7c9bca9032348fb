"""Calls of the bounded cache that are refused leave everything as it was."""
import numpy as np
import pytest

from test_gpu_bounded import BS, kv, make  # noqa: F401 (kv is the module's fixture)
from test_gpu_evict import want_keep

pytestmark = pytest.mark.gpu


def shared(kv, spare):
    """Two sequences of 96 rows over the same six blocks, `spare` blocks free; (cache, tokens)."""
    c = make(kv, [96, 0], True, 2, spare=spare)
    t = np.arange(96, dtype=np.uint32)
    prefix = kv.NO_HASH
    for bi in range(6):
        c.seq_cache_block(0, bi, t[bi * BS:(bi + 1) * BS], prefix)
        prefix = kv.KVCache.computeHash(t[bi * BS:(bi + 1) * BS], prefix)
    c.seq_reuse_prefix_blocks(1, t, 6)
    assert c.numFreeBlocks() == spare
    return c, t


def state(c, t):
    tables = [c.seq_block_table(s) for s in range(2)]
    return (tables, [c.refcount(b) for b in range(c.num_blocks)], c.numFreeBlocks(), c.findPrefixBlocks(t),
            [c.seq_len(s) for s in range(2)], [c.gather(layer, s).tobytes() for layer in range(2) for s in range(2)])


@pytest.mark.parametrize("ids,needed", [([1], 4), ([0, 1], 4), ([1, 0], 4)])
def test_too_few_blocks_for_the_copies(kv, ids, needed):
    """One of the two holders moves its rows in copies, or both do: the second has the blocks for itself."""
    import torch

    c, t = shared(kv, needed - 1)
    before = state(c, t)
    mass = torch.rand(2, len(ids), 96, device="cuda")
    kept = mass.clone()
    with pytest.raises(kv.KVCudaError) as e:
        c.evict_dev(ids, 64, mass)
    assert e.value.name == "OutOfKVCacheBlocks"
    assert state(c, t) == before and before[3] == 6 and torch.equal(mass, kept)


@pytest.mark.parametrize("ids", [[1], [0, 1], [1, 0]])
def test_just_enough_blocks_for_the_copies(kv, ids):
    import torch

    c, t = shared(kv, 4)
    rows = [[c.gather(layer, s) for s in range(2)] for layer in range(2)]
    mass = torch.rand(2, len(ids), 96, device="cuda")
    m = mass.cpu().numpy()
    c.evict_dev(ids, 64, mass, 3, 5)
    assert c.pool().status() == 0
    for layer in range(2):
        for s in range(2):
            want = rows[layer][s]
            if s in ids:
                want = want[want_keep(m[layer, ids.index(s)], 96, 64, 3, 5)]
            assert np.array_equal(c.gather(layer, s), want)
    # the blocks that still hold the prefix are those of the sequence that stayed
    assert c.findPrefixBlocks(t) == (0 if len(ids) == 2 else 6)
    live = {b for s in range(2) for b in c.seq_block_table(s)}
    assert c.numFreeBlocks() + len(live) == c.num_blocks
