"""kvcu_evict_select and kvcu_evict_compact on the GPU: the choice against a sort,
the moved rows byte for byte against the same moves on a copy of the pool."""
import numpy as np
import pytest

from pooldata import Paged, arrays

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    import torch

    import kvcu

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    kvcu.init(0)
    return kvcu


def want_keep(mass, length, budget, sink, recent):
    """The kept positions of one row: the ends, then by (value descending, position), NaN last."""
    if length <= budget:
        return np.arange(length)
    mid = mass[sink:length - recent].astype(np.float64)
    rank = np.where(np.isnan(mid), 0, 1)
    order = np.lexsort((np.arange(len(mid)), -np.where(np.isnan(mid), 0, mid), -rank))
    chosen = sink + np.sort(order[:budget - sink - recent])
    return np.concatenate([np.arange(sink), chosen, np.arange(length - recent, length)])


def select(kv, pool, mass, lens, budget, sink, recent, wide=0, seq_ids=None):
    import torch

    nl, n = mass.shape[:2]
    keep = torch.full((nl, n, budget + wide), 12345, dtype=torch.int32, device="cuda")
    counts = torch.full((n,), 12345, dtype=torch.int32, device="cuda")
    pool.evict_select(mass, lens, budget, sink, recent, keep, counts, seq_ids=seq_ids)
    return keep, counts


def check_select(kv, pool, mass, lens, budget, sink, recent, wide=0, rows=None):
    import torch

    lens_dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    keep, counts = select(kv, pool, mass, lens_dev, budget, sink, recent, wide)
    assert pool.status() == 0
    m, k, c = mass.cpu().numpy(), keep.cpu().numpy(), counts.cpu().numpy()
    for b, length in enumerate(lens):
        assert c[b] == min(length, budget)
        for layer in range(m.shape[0]):
            want = want_keep(m[layer, b], length, budget, sink, recent)
            assert np.array_equal(k[layer, b, :c[b]], want), (layer, b, length)
            assert (k[layer, b, c[b]:budget] == -1).all()
            assert (k[layer, b, budget:] == 12345).all()


@pytest.fixture(scope="module")
def pool(kv):
    return kv.DevicePool(0, 1, 1, 16, 512, 64, True)


def _mass(kind, shape, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if kind == "heavy":  # log-normal, a tenth zeros
        x = (x * 3).exp()
        x[torch.rand(shape, generator=g, device="cuda") < 0.1] = 0
    elif kind == "ties":
        x = (x * 2).round()
        x[x == 0] = torch.where(torch.rand(int((x == 0).sum()), generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif kind == "equal":
        x = torch.full(shape, 0.25, device="cuda")
    elif kind == "special":
        r = torch.rand(shape, generator=g, device="cuda")
        x[r < 0.2] = float("nan")
        x[(r > 0.2) & (r < 0.3)] = float("inf")
        x[(r > 0.3) & (r < 0.4)] = float("-inf")
        x[(r > 0.4) & (r < 0.5)] = 1e-42
        x[(r > 0.5) & (r < 0.6)] = -1e-42
    return x


@pytest.mark.parametrize("kind", ["plain", "heavy", "ties", "equal", "special"])
@pytest.mark.parametrize("layers,lens,budget,sink,recent", [
    (1, [0, 1, 2, 31, 32, 33, 64, 65], 32, 0, 0),
    (2, [100, 63, 64, 65, 1000, 999], 64, 4, 16),
    (3, [5000, 4097, 129, 12000], 128, 0, 128),
    (1, [40, 41, 2000], 40, 40, 0),
    (1, [40, 41, 2000], 40, 10, 30),
    (2, [9000], 1, 0, 0),
    (1, [9000, 8999], 8998, 1, 2),
])
def test_select(kv, pool, kind, layers, lens, budget, sink, recent):
    check_select(kv, pool, _mass(kind, (layers, len(lens), max(lens) + 3), 11), lens, budget, sink, recent, wide=2)


@pytest.mark.parametrize("kind", ["heavy", "ties"])
def test_select_long_rows_in_clusters(kv, pool, kind):
    """Rows shared by 2, 4 and 8 CTAs, and rows longer than the shared memory of eight."""
    check_select(kv, pool, _mass(kind, (1, 200, 49500), 1), [49500 - 7 * i for i in range(200)], 1500, 16, 64)
    check_select(kv, pool, _mass(kind, (1, 40, 20001), 1), [20001 - 100 * i for i in range(40)], 777, 3, 5)
    check_select(kv, pool, _mass(kind, (2, 5, 70000), 2), [70000, 69999, 300, 30000, 65536], 4096, 4, 256)
    check_select(kv, pool, _mass(kind, (1, 2, 430001), 3), [430001, 400000], 5000, 16, 100)
    check_select(kv, pool, _mass(kind, (1, 2, 430001), 3), [430001, 5001], 429000, 0, 100)


def test_select_chosen_sequences_and_bad_ones(kv, pool):
    import torch

    mass = _mass("plain", (2, 3, 500), 4)
    lens = torch.tensor([500, 20, 300, 400], dtype=torch.int32, device="cuda")
    ids = torch.tensor([3, 0, 2], dtype=torch.int32, device="cuda")
    keep, counts = select(kv, pool, mass, lens, 64, 2, 8, seq_ids=ids)
    assert pool.status() == 0
    for b, length in enumerate([400, 500, 300]):
        for layer in range(2):
            assert np.array_equal(keep[layer, b].cpu().numpy(), want_keep(mass[layer, b].cpu().numpy(), length, 64, 2, 8))
    ids[1] = 9
    keep, counts = select(kv, pool, mass, lens, 64, 2, 8, seq_ids=ids)
    assert pool.status() == 0x4 and counts.tolist() == [64, 0, 64] and (keep[:, 1] == -1).all()
    lens += 100  # beyond the rows of sums: cut
    ids[1] = 0
    keep, counts = select(kv, pool, mass, lens, 64, 2, 8, seq_ids=ids)
    assert pool.status() == 0x8
    assert np.array_equal(keep[0, 1].cpu().numpy(), want_keep(mass[0, 1].cpu().numpy(), 500, 64, 2, 8))


def test_select_refusals(kv, pool):
    import torch

    mass, lens = torch.zeros(1, 2, 100, device="cuda"), torch.tensor([100, 100], dtype=torch.int32, device="cuda")
    for budget, sink, recent in ((0, 0, 0), (10, 6, 5), (10, 11, 0)):
        with pytest.raises(kv.KVCudaError) as e:
            select(kv, pool, mass, lens, budget, sink, recent)
        assert e.value.name == "InvalidArgument"
    keep, counts = torch.zeros(1, 2, 10, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pool.evict_select(mass, lens, 11, 0, 0, keep, counts)
    with pytest.raises(ValueError):
        pool.evict_select(mass, lens, 5, 0, 0, keep, counts[:1])
    with pytest.raises(ValueError):
        pool.evict_select(mass[:, :, ::2], lens, 5, 0, 0, keep, counts)
    with pytest.raises(ValueError):
        pool.evict_select(mass, lens[:1], 5, 0, 0, keep, counts)


def _keep_lists(rng, layers, lens, budget, kind):
    keep = np.full((layers, len(lens), budget), -1, np.int32)
    counts = [min(x, budget) for x in lens]
    for layer in range(layers):
        for b, length in enumerate(lens):
            c = counts[b]
            if kind == "random":
                k = np.sort(rng.choice(length, c, replace=False))
            elif kind == "last":
                k = np.arange(length - c, length)
            elif kind == "alternate":
                k = np.unique(np.minimum(np.arange(c) * 2, length - c + np.arange(c)))
            else:  # the first ones, then one hole
                k = np.arange(c) + (np.arange(c) >= c // 2) * (1 if length > c else 0)
            keep[layer, b, :c] = k
    return keep, counts


@pytest.mark.parametrize("kind", ["random", "last", "alternate", "hole"])
@pytest.mark.parametrize("quant,dims,bs,layers,lens,budget", [
    (True, (512, 64), 64, 2, [700, 64, 100, 3000, 1, 0], 100),
    (True, (512, 64), 16, 1, [5000], 2047),
    (True, (512, 64), 16, 8, [640], 512),
    (False, (512, 64), 16, 2, [500, 129], 77),
    (True, (16, 8), 16, 2, [100, 40], 33),
    (False, (16, 8), 16, 2, [100, 40], 33),
    (False, (6, 10), 32, 1, [300], 100),
    (True, (33, 64), 32, 1, [300, 200], 64),
    (True, (96, 32), 48, 3, [333, 47], 48),
    (True, (32, 64), 16, 2, [300, 77], 60),
    (False, (128, 24), 16, 2, [300, 77], 60),
    (False, (12, 8), 16, 1, [300], 160),
])
def test_compact(kv, kind, quant, dims, bs, layers, lens, budget):
    import torch

    rng = np.random.default_rng(budget)
    cache = Paged(kv, lens, bs, quant, layers=layers + 1, seed=3, dims=dims)
    keep, counts = _keep_lists(rng, layers, lens, budget, kind)
    want = [x.cpu().numpy().copy() for x in arrays(cache.pool)]
    mass = torch.rand(layers, len(lens), max(lens) + 2, device="cuda")
    wmass = mass.cpu().numpy().copy()
    for layer in range(layers):
        for b in range(len(lens)):
            k = keep[layer, b, :counts[b]].astype(np.int64)
            to, at = cache.rows_at(b, np.arange(counts[b]), layer + 1), cache.rows_at(b, k, layer + 1)
            for x in want:
                x[to] = x[at]
            wmass[layer, b, :counts[b]] = wmass[layer, b, k]
    lens_dev = cache.lens_dev.clone()
    cache.pool.evict_compact(1, cache.toff, cache.tables, torch.from_numpy(keep).cuda(),
                             torch.tensor(counts, dtype=torch.int32, device="cuda"), mass=mass, lens=lens_dev)
    assert cache.pool.status() == 0
    for got, w in zip(arrays(cache.pool), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert np.array_equal(mass.cpu().numpy(), wmass)
    assert lens_dev.tolist() == counts


def test_compact_many_pairs_and_long_lists(kv):
    """More pairs than the grid has room for clusters, and lists of many waves."""
    import torch

    rng = np.random.default_rng(5)
    lens = [2500 + 37 * i for i in range(40)]
    cache = Paged(kv, lens, 64, True, layers=4, seed=6)
    keep, counts = _keep_lists(rng, 4, lens, 2000, "random")
    want = [x.cpu().numpy().copy() for x in arrays(cache.pool)]
    for layer in range(4):
        for b in range(40):
            to, at = (cache.rows_at(b, p, layer) for p in (np.arange(2000), keep[layer, b]))
            for x in want:
                x[to] = x[at]
    cache.pool.evict_compact(0, cache.toff, cache.tables, torch.from_numpy(keep).cuda(),
                             torch.tensor(counts, dtype=torch.int32, device="cuda"))
    for got, w in zip(arrays(cache.pool), want):
        assert np.array_equal(got.cpu().numpy(), w)


def test_compact_chosen_sequences_and_bad_entries(kv):
    import torch

    cache = Paged(kv, [200, 300, 400], 16, True, seed=7)
    ids = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    keep = np.stack([np.arange(100) * 3, np.arange(100) * 2])[None].astype(np.int32)
    counts = torch.tensor([100, 100], dtype=torch.int32, device="cuda")
    want = [x.cpu().numpy().copy() for x in arrays(cache.pool)]
    for b, s in enumerate([2, 0]):
        to, at = cache.rows_at(s, np.arange(100)), cache.rows_at(s, keep[0, b])
        for x in want:
            x[to] = x[at]
    lens = cache.lens_dev.clone()
    cache.pool.evict_compact(0, cache.toff, cache.tables, torch.from_numpy(keep).cuda(), counts, lens=lens, seq_ids=ids)
    assert cache.pool.status() == 0 and lens.tolist() == [100, 300, 100]
    for got, w in zip(arrays(cache.pool), want):
        assert np.array_equal(got.cpu().numpy(), w)
    # a position behind the table and a block behind the pool: their rows are left, the others move
    cache = Paged(kv, [200], 16, True, seed=8)
    keep = (np.arange(50) * 2 + 10)[None, None].astype(np.int32)
    keep[0, 0, 49] = 100000
    tables = cache.tables.clone()
    tables[2] = cache.nb + 5  # positions 32..47
    want = [x.cpu().numpy().copy() for x in arrays(cache.pool)]
    ok = [j for j in range(49) if not 32 <= j < 48 and not 32 <= keep[0, 0, j] < 48]
    to, at = cache.rows_at(0, np.array(ok)), cache.rows_at(0, keep[0, 0, ok])
    for x in want:
        x[to] = x[at]
    cache.pool.evict_compact(0, cache.toff, tables, torch.from_numpy(keep).cuda(),
                             torch.tensor([50], dtype=torch.int32, device="cuda"))
    assert cache.pool.status() == 0x3
    for got, w in zip(arrays(cache.pool), want):
        assert np.array_equal(got.cpu().numpy(), w)


def test_compact_refusals(kv):
    import torch

    cache = Paged(kv, [200], 16, True, layers=2, seed=8)
    keep = torch.zeros(1, 1, 10, dtype=torch.int32, device="cuda")
    counts = torch.ones(1, dtype=torch.int32, device="cuda")
    for layer, k in ((2, keep), (1, keep.expand(2, 1, 10).contiguous())):
        with pytest.raises(kv.KVCudaError) as e:
            cache.pool.evict_compact(layer, cache.toff, cache.tables, k, counts)
        assert e.value.name == "LayerOutOfBounds"
    with pytest.raises(ValueError):
        cache.pool.evict_compact(0, cache.toff, cache.tables, keep.expand(1, 2, 10).contiguous(), counts)
    with pytest.raises(ValueError):
        cache.pool.evict_compact(0, cache.toff, cache.tables, keep, counts, mass=torch.zeros(2, 1, 10, device="cuda"))


def test_select_then_compact_in_a_graph(kv):
    """The two calls captured once and replayed on other sums."""
    import torch

    cache = Paged(kv, [900, 300], 64, True, layers=2, seed=9)
    mass = _mass("heavy", (2, 2, 900), 1)
    keep = torch.empty(2, 2, 128, dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):  # set-up outside the capture
        cache.pool.evict_select(mass, cache.lens_dev, 128, 4, 16, keep, counts, stream=s)
        cache.pool.evict_compact(0, cache.toff, cache.tables, keep, torch.zeros_like(counts), stream=s)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream()
        cache.pool.evict_select(mass, cache.lens_dev, 128, 4, 16, keep, counts, stream=st)
        cache.pool.evict_compact(0, cache.toff, cache.tables, keep, counts, mass=mass, stream=st)
    mass.copy_(_mass("heavy", (2, 2, 900), 2))
    m = mass.cpu().numpy().copy()
    want = [x.cpu().numpy().copy() for x in arrays(cache.pool)]
    for layer in range(2):
        for b in range(2):
            k = want_keep(m[layer, b], cache.lens[b], 128, 4, 16)
            for x in want:
                x[cache.rows_at(b, np.arange(128), layer)] = x[cache.rows_at(b, k, layer)]
            m[layer, b, :128] = m[layer, b, k]
    graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(arrays(cache.pool), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert np.array_equal(mass.cpu().numpy(), m)
