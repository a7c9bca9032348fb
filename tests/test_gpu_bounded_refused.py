"""Calls of the bounded cache that are refused leave everything as it was."""
import numpy as np
import pytest

from kvdata import SCALE
from pooldata import Paged, arrays
from test_gpu_bounded import BS, Cached, P, R, Step, kv, make  # noqa: F401 (kv is the module's fixture)
from test_gpu_evict import want_keep
from test_gpu_mass import check, want_mass

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


def compact(kv, cache, keep, counts, mass, layer_stride, stride):
    """The C call, with any strides of the sums."""
    layers, n, budget = keep.shape
    return kv.lib().kvcu_evict_compact(cache.pool.handle, 0, layers, n, None, n, cache.toff.data_ptr(),
                                       cache.tables.data_ptr(), keep.data_ptr(), n * budget, budget, counts.data_ptr(),
                                       mass.data_ptr(), layer_stride, stride, None, None)


def test_rows_of_sums_that_overlap(kv):
    """All rows of sums move at once, so no two may share one."""
    import torch

    cache = Paged(kv, [200, 200, 200], 16, True, layers=2, seed=4)
    before = [x.clone() for x in arrays(cache.pool)]
    keep = torch.arange(100, dtype=torch.int32, device="cuda").mul_(2).repeat(2, 3, 1)
    counts = torch.full((3,), 100, dtype=torch.int32, device="cuda")
    mass = torch.rand(2, 3, 200, device="cuda")
    kept = mass.clone()
    # no layers apart, no entries apart, no row between, layers inside the entries, entries inside the layers
    for strides in ((0, 200), (600, 0), (0, 0), (200, 200), (400, 200), (200, 100), (2 ** 63, 2 ** 63)):
        assert compact(kv, cache, keep, counts, mass, *strides) == -11, strides
    with pytest.raises(kv.KVCudaError):
        cache.pool.evict_compact(0, cache.toff, cache.tables, keep, counts, mass=mass[:1].expand(2, 3, 200))
    c, _ = shared(kv, 8)
    for strides in ((0, 96), (96, 96), (96, 0)):
        ids = np.array([0, 1], np.uint32)
        assert kv.lib().kvcache_evict_dev(c._h, 2, ids.ctypes.data, 64, 0, 0, mass.data_ptr(), *strides, None, None) == -11
    assert c.seq_len(0) == 96 and c.numFreeBlocks() == 8
    torch.cuda.synchronize()
    assert torch.equal(mass, kept) and all(torch.equal(a, b) for a, b in zip(arrays(cache.pool), before))


def test_sums_of_empty_sequences_may_have_no_room(kv):
    import torch

    c = make(kv, [0, 0], True, 2)
    ids, some = np.array([0, 1], np.uint32), torch.zeros(1, device="cuda")
    assert kv.lib().kvcache_evict_dev(c._h, 2, ids.ctypes.data, 8, 0, 0, some.data_ptr(), 0, 0, None, None) == 0
    assert c.last_launches == 0 and c.seq_len(0) == 0


def test_sums_with_the_layers_inside_the_entries(kv):
    """[entry][layer][position] is a layout of its own, and one entry's rows may be any distance apart."""
    import torch

    for n in (3, 1):
        cache = Paged(kv, [200] * n, 16, True, layers=2, seed=4)
        keep = torch.arange(100, dtype=torch.int32, device="cuda").mul_(2).repeat(2, n, 1)
        counts = torch.full((n,), 100, dtype=torch.int32, device="cuda")
        mass = torch.rand(n, 2, 200, device="cuda")
        want = mass.clone()
        want[:, :, :100] = mass[:, :, :200:2]
        assert compact(kv, cache, keep, counts, mass, 200, 400) == 0
        assert cache.pool.status() == 0 and torch.equal(mass, want)


@pytest.mark.parametrize("dims", [(512, 64), (64, 32)])  # rows moved through registers, and through shared memory
def test_a_kept_position_beyond_its_row_of_sums(kv, dims):
    import torch

    cache = Paged(kv, [200], 16, True, layers=2, seed=4, dims=dims)
    keep = torch.arange(100, dtype=torch.int32, device="cuda").mul_(2).repeat(2, 1, 1)
    counts = torch.full((1,), 100, dtype=torch.int32, device="cuda")
    mass = torch.rand(2, 1, 150, device="cuda") + 1
    want = mass.clone()
    want[:, :, :75] = mass[:, :, ::2]
    want[:, :, 75:100] = 0
    cache.pool.evict_compact(0, cache.toff, cache.tables, keep, counts, mass=mass)
    assert cache.pool.status() == 0x8 and torch.equal(mass, want)


def test_weights_of_a_sequence_that_a_load_took_away(kv, tmp_path):
    """The step's plan still lists it; the cache has one sequence left."""
    import torch

    c = make(kv, [40, 20, 30], True, 1)
    one = kv.KVCache.with_blocks(1, R, P, c.num_blocks, BS, quantized=True)
    one.saveToFileV2(tmp_path / "one.ckpt")
    st = Step(2, 6)
    c.seq_ensure_capacity(0, 41), c.seq_ensure_capacity(2, 31)
    st.run(c, 0, [0, 2], [40, 30], kv.Rope(P))
    c.loadFromFileV2(tmp_path / "one.ckpt")
    mass = torch.ones(2, 64, device="cuda")
    with pytest.raises(kv.KVCudaError) as e:
        c.attnMass_dev(0, [0, 2], st.q_abs, st.lse, SCALE, mass)
    assert e.value.name == "InvalidArgument" and "sequence 2 does not exist" in str(e.value)
    torch.cuda.synchronize()
    assert (mass == 1).all() and c.pool().status() == 0


def test_weights_after_a_refused_step_of_a_larger_cache(kv):
    """The refused step needed more room for its ids; the plan of the step before goes by its own."""
    import torch

    lens = [40, 20]
    c = make(kv, lens, True, 1)
    st = Step(2, 6)
    for s in range(2):
        c.seq_ensure_capacity(s, lens[s] + 1)
    st.run(c, 0, [0, 1], lens, kv.Rope(P))
    for _ in range(5000):
        c.seq_create()
    with pytest.raises(kv.KVCudaError):
        Step(2, 7).run(c, 0, [0, 0], [41, 41], kv.Rope(P))
    lens = [41, 21]
    before = torch.ones(2, 64, device="cuda")
    mass = before.clone()
    c.attnMass_dev(0, [0, 1], st.q_abs, st.lse, SCALE, mass)
    assert c.pool().status() == 0
    want, tol = want_mass(Cached(c, lens), [0, 1], st.q_abs[:, None], st.lse[:, None], before, 1.0, lens)
    check(mass, want, tol)


def test_on_a_stream_that_is_being_captured(kv):
    """The cache's calls keep state on the host, which a graph would not repeat."""
    import torch

    c, t = shared(kv, 8)
    st, rope = Step(1, 6), kv.Rope(P)
    mass, keep = torch.rand(2, 1, 96, device="cuda"), torch.empty(2, 1, 96, dtype=torch.int32, device="cuda")
    c.evict_dev([1], 96, mass, keep_dev=keep)  # within the budget: kernels loaded, scratch there
    before, kept = state(c, t), mass.clone()
    c.seq_truncate(1, 95)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream()
        for f in (lambda: c.evict_dev([1], 64, mass, stream=s), lambda: c.evict_dev([0], 64, mass, keep_dev=keep[:, :, :64].contiguous(), stream=s),
                  lambda: c.attnMass_dev(0, [1], st.q_abs, st.lse, SCALE, mass[0], old_lens=[95], stream=s),
                  lambda: st.run(c, 0, [1], [95], rope, stream=s)):
            with pytest.raises(kv.KVCudaError) as e:
                f()
            assert e.value.name == "Unsupported", e.value
    del graph
    st.run(c, 0, [0], [95], rope)
    assert c.seq_len(0) == 96 and c.seq_len(1) == 95
    assert [c.seq_block_table(s) for s in range(2)] != before[0]  # the step copied the block it wrote into
    assert torch.equal(mass, kept)
    c.evict_dev([1], 64, mass)
    assert c.seq_len(1) == 64 and c.pool().status() == 0
