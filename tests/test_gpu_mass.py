"""kvcu_attn_mass on the GPU against the sums in 64 bits.

Tolerances.  A score is a sum of 576 products in f32 (or of exact f16 parts of q, 22
bits, against exact int8 values): each position's score is off by at most
(160 + 4) * 2^-24 * scale * sum |q k|, its weight by that much relative to itself plus
the roundings of the exponent's argument and of expf (a few 2^-24 of |s| + |lse| + 1);
the sum over queries and heads adds (n_q * heads + 2) * 2^-24.  That is the bound of
every position.  Roundings have either sign, so the 2-norm of all errors is far
smaller: sqrt(576) * 2^-24 * |s|, under 4e-6."""
import math

import numpy as np
import pytest

from pooldata import Paged, W

pytestmark = pytest.mark.gpu
SCALE = 1.0 / math.sqrt(192.0)


@pytest.fixture(scope="module")
def kv():
    import torch

    import kvcu

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    kvcu.init(0)
    return kvcu


def queries(cache, seqs, n_q, heads, seed, layer=0, lens=None, spread=0.05):
    """q [n][n_q][heads][W] and its log-sum-exp over what each query sees (f32 of 64 bits)."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    n = len(seqs)
    q = torch.randn(n, n_q, heads, W, device="cuda", generator=g) * spread
    lse = torch.full((n, n_q, heads), -math.inf, device="cuda")
    for b, s in enumerate(seqs):
        length = cache.lens[s] if lens is None else lens[b]
        k = cache.values(s, layer)[:length]
        for i in range(n_q):
            seen = length - (n_q - 1 - i)
            if seen > 0:
                lse[b, i] = torch.logsumexp(q[b, i].double() @ k[:seen].T * SCALE, 1).float()
    return q, lse


def want_mass(cache, seqs, q, lse, mass, decay, old, layer=0, lens=None):
    """(mass in 64 bits, bound of each position's error); positions behind the length: mass itself, 0."""
    import torch

    out, tol = mass.double().clone(), torch.zeros_like(mass, dtype=torch.float64)
    u = 2.0 ** -24
    n_q, heads = q.shape[1], q.shape[2]
    for b, s in enumerate(seqs):
        length = cache.lens[s] if lens is None else lens[b]
        k = cache.values(s, layer)[:length]
        total, err = torch.zeros(length, device="cuda", dtype=torch.float64), torch.zeros(length, device="cuda",
                                                                                         dtype=torch.float64)
        for i in range(n_q):
            seen = length - (n_q - 1 - i)
            if seen <= 0:
                continue
            qi, l = q[b, i].double(), lse[b, i].double()[:, None]
            sc = qi @ k[:seen].T * SCALE
            w = torch.exp(sc - l)
            es = 164 * u * SCALE * (qi.abs() @ k[:seen].abs().T) + 4 * u * (sc.abs() + l.abs() + 1)
            total[:seen] += w.sum(0)
            err[:seen] += (w * es * 1.01).sum(0)
        err += (n_q * heads + 2) * u * total
        before = torch.where(torch.arange(length, device="cuda") < old[b], decay * mass[b, :length].double(),
                             torch.zeros(length, device="cuda", dtype=torch.float64))
        out[b, :length] = before + total
        tol[b, :length] = err + 2 * u * (before.abs() + total)
    return out, tol


def check(got, want, tol):
    import torch

    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())
    live = tol > 0
    assert (err[live].norm() <= 4e-6 * want[live].norm()), float(err[live].norm() / want[live].norm())


LENS = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, 2000, 5001]


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("heads,bs", [(20, 64), (1, 16), (7, 48), (8, 128), (9, 16), (16, 256), (17, 32), (24, 64), (25, 16),
                                      (32, 64)])
def test_step(kv, quant, heads, bs):
    import torch

    cache = Paged(kv, LENS, bs, quant, layers=2, seed=heads)
    n = len(LENS)
    q, lse = queries(cache, range(n), 1, heads, 7, layer=1)
    longest = max(LENS) + 5
    mass = torch.rand(n, longest, device="cuda")
    old = torch.tensor([max(0, x - 1) for x in LENS], dtype=torch.int32, device="cuda")
    want, tol = want_mass(cache, range(n), q, lse, mass, 0.9, old, layer=1)
    behind = mass.clone()
    ws = kv.DecodeWorkspace(0, n, heads)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 1, q[:, 0].contiguous(), lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, decay=0.9,
                 old_lens=old)
    assert cache.pool.status() == 0
    check(mass, want, tol)
    for b, length in enumerate(LENS):
        assert torch.equal(mass[b, length:], behind[b, length:])


@pytest.mark.parametrize("quant,n_q,heads,bs", [(True, 2, 20, 64), (True, 33, 20, 16), (False, 5, 8, 16), (True, 7, 32, 64),
                                                (True, 3, 8, 48), (False, 4, 20, 64)])
def test_window_of_queries(kv, quant, n_q, heads, bs):
    """Several queries per entry, each with its own limit; entries shorter than the window, where
    the first queries see nothing."""
    import torch

    lens = [1, 3, n_q - 1, n_q, n_q + 1, 64 + n_q, 900, 1601]
    cache = Paged(kv, lens, bs, quant, seed=n_q)
    n = len(lens)
    q, lse = queries(cache, range(n), n_q, heads, 3)
    mass = torch.rand(n, max(lens), device="cuda")
    want, tol = want_mass(cache, range(n), q, lse, mass, 1.0, lens)
    ws = kv.DecodeWorkspace(0, n, heads)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass)
    assert cache.pool.status() == 0
    check(mass, want, tol)


@pytest.mark.parametrize("quant", [True, False])
def test_chosen_sequences_grown_since_the_plan(kv, quant):
    """A batch of some sequences, one of them twice, planned when they were shorter."""
    import torch

    cache = Paged(kv, [300, 5000, 64, 900], 64, quant, seed=9)
    seqs = [3, 1, 1, 0]
    ids = torch.tensor(seqs, dtype=torch.int32, device="cuda")
    q, lse = queries(cache, seqs, 1, 20, 4)
    mass = torch.rand(4, 5000, device="cuda")
    want, tol = want_mass(cache, seqs, q, lse, mass, 0.5, [cache.lens[s] for s in seqs])
    ws = kv.DecodeWorkspace(0, 8, 20)
    ws.plan(cache.pool, torch.clamp(cache.lens_dev - 40, min=0), seq_ids=ids)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, decay=0.5, seq_ids=ids)
    check(mass, want, tol)


def test_causal_plan(kv):
    """Entries of one sequence with lengths of their own (a causal plan): each has its own sums."""
    import ctypes as C

    import torch

    cache = Paged(kv, [700], 64, True, seed=2)
    el = [1, 64, 500, 700]
    seqs = [0] * 4
    q, lse = queries(cache, seqs, 1, 20, 4, lens=el)
    mass = torch.rand(4, 700, device="cuda")
    want, tol = want_mass(cache, seqs, q, lse, mass, 1.0, el, lens=el)
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    eld = torch.tensor(el, dtype=torch.int32, device="cuda")
    ws = kv.DecodeWorkspace(0, 4, 20)
    assert kv.lib().kvcu_decode_plan_causal(ws._h, cache.pool.handle, 4, ids.data_ptr(), 1, cache.lens_dev.data_ptr(),
                                            eld.data_ptr(), None) == 0
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, seq_ids=ids)
    check(mass, want, tol)


def test_weights_of_one_step_sum_to_the_heads(kv):
    """With the log-sum-exp of the product's own decode, every head's weights sum to 1."""
    import torch

    cache = Paged(kv, [777, 3000], 64, True, seed=3)
    heads = 20
    q = torch.randn(2, heads, W, device="cuda") * 0.05
    out, lse = torch.empty(2, heads, 512, device="cuda"), torch.empty(2, 1, heads, device="cuda")
    ws = kv.DecodeWorkspace(0, 2, heads)
    ws.plan(cache.pool, cache.lens_dev)
    assert kv.lib().kvcu_mla_decode_lse(ws._h, cache.pool.handle, 0, 2, None, 2, cache.toff.data_ptr(),
                                        cache.tables.data_ptr(), cache.lens_dev.data_ptr(), q.data_ptr(), heads, SCALE,
                                        out.data_ptr(), lse.data_ptr(), None) == 0
    mass = torch.zeros(2, 3000, device="cuda")
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass)
    # the decode's scores round q to two int8 digits: its lse is within its 1e-3 attention tolerance
    assert (mass.sum(1) / heads - 1).abs().max() <= 1e-3


@pytest.mark.parametrize("scale_q", [1e-20, 1e-4, 300.0, 1e5])
def test_far_ranges_of_q(kv, scale_q):
    """Queries far from 1: the scores are brought back to ordinary size by the scale."""
    import torch

    cache = Paged(kv, [300, 129], 64, True, seed=4)
    q, _ = queries(cache, [0, 1], 1, 20, 6)
    qs, scale = (q * scale_q).contiguous(), SCALE / scale_q
    lse = torch.empty(2, 1, 20, device="cuda")
    want = torch.zeros(2, 300, dtype=torch.float64, device="cuda")
    for b in range(2):
        s = qs[b, 0].double() @ cache.values(b).T * scale
        lse[b, 0] = torch.logsumexp(s, 1).float()
        want[b, :cache.lens[b]] = torch.exp(s - lse[b, 0].double()[:, None]).sum(0)
    mass = torch.zeros(2, 300, device="cuda")
    ws = kv.DecodeWorkspace(0, 2, 20)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 0, qs, lse, cache.toff, cache.tables, cache.lens_dev, scale, mass)
    # the bound of the file's head with these rows: scale * sum |q k| < 6, |s| + |lse| < 20
    assert (mass.double() - want).abs().max() <= 2e-4 * want.abs().max()
    assert (mass.double() - want).norm() <= 4e-6 * want.norm()


def test_same_bits_twice_and_in_a_graph(kv):
    import torch

    cache = Paged(kv, [5000, 64, 900, 1], 64, True, seed=5)
    q, lse = queries(cache, range(4), 1, 20, 6)
    ws = kv.DecodeWorkspace(0, 4, 20)
    ws.plan(cache.pool, cache.lens_dev)
    old = torch.zeros(4, dtype=torch.int32, device="cuda")
    masses = [torch.full((4, 5000), float("nan"), device="cuda") for _ in range(3)]  # new sums read nothing old
    for m in masses[:2]:
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, m, old_lens=old)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, masses[2], old_lens=old,
                     stream=torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    for b in range(4):
        a = masses[0][b, :cache.lens[b]]
        assert torch.isfinite(a).all()
        assert torch.equal(a, masses[1][b, :cache.lens[b]]) and torch.equal(a, masses[2][b, :cache.lens[b]])
        assert torch.isnan(masses[0][b, cache.lens[b]:]).all()


def test_bad_blocks_and_lengths_set_the_status(kv):
    import torch

    cache = Paged(kv, [200, 300], 16, True, seed=6)
    q, lse = queries(cache, range(2), 1, 20, 6)
    mass = torch.rand(2, 300, device="cuda")
    want, tol = want_mass(cache, range(2), q, lse, mass, 1.0, cache.lens)
    before = mass.clone()
    tables = cache.tables.clone()
    tables[3] = cache.nb  # positions 48..63 of sequence 0
    ws = kv.DecodeWorkspace(0, 2, 20)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, tables, cache.lens_dev, SCALE, mass)
    assert cache.pool.status() == 0x2
    assert torch.equal(mass[0, 48:64], before[0, 48:64])
    mass[0, 48:64] = want[0, 48:64].float()
    check(mass, want, tol)
    # a length beyond the table is cut to it, one beyond the row of sums as well
    long = cache.lens_dev + 100
    mass = before.clone()
    ws.plan(cache.pool, long)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, long, SCALE, mass)
    assert cache.pool.status() == 0x8
    short = before[:, :150].contiguous()
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, short)
    assert cache.pool.status() == 0x8
    assert ((short.double() - want[:, :150]).abs() <= tol[:, :150]).all()
    ids = torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    ws.plan(cache.pool, cache.lens_dev, seq_ids=ids)
    mass = before.clone()
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, seq_ids=ids)
    assert cache.pool.status() in (0, 0x4)  # the planned entry has no tokens: it may have no work at all
    assert torch.equal(mass[1], before[1])


def test_refusals(kv):
    import torch

    cache = Paged(kv, [100, 50], 16, True, seed=8)
    q, lse = queries(cache, range(2), 1, 20, 6)
    mass = torch.zeros(2, 100, device="cuda")
    args = (cache.toff, cache.tables, cache.lens_dev, SCALE)
    ws = kv.DecodeWorkspace(0, 4, 20, max_layers=2)
    with pytest.raises(kv.KVCudaError) as e:  # no plan yet
        ws.attn_mass(cache.pool, 0, q, lse, *args, mass)
    assert e.value.name == "InvalidArgument"
    ws.plan(cache.pool, cache.lens_dev)
    with pytest.raises(kv.KVCudaError) as e:
        ws.attn_mass(cache.pool, 1, q, lse, *args, mass)
    assert e.value.name == "LayerOutOfBounds"
    with pytest.raises(kv.KVCudaError):  # another batch than the plan's
        ws.attn_mass(cache.pool, 0, q[:1].contiguous(), lse[:1].contiguous(), *args, mass[:1])
    with pytest.raises(kv.KVCudaError) as e:
        ws.attn_mass(cache.pool, 0, torch.zeros(2, 33, W, device="cuda"), torch.zeros(2, 33, device="cuda"), *args, mass)
    assert e.value.name == "Unsupported"
    with pytest.raises(ValueError):
        ws.attn_mass(cache.pool, 0, q, lse[:, :, :19], *args, mass)
    with pytest.raises(ValueError):
        ws.attn_mass(cache.pool, 0, q, lse, *args, torch.zeros(3, 100, device="cuda"))
    with pytest.raises(ValueError):
        ws.attn_mass(cache.pool, 0, q, lse, *args, torch.zeros(2, 200, device="cuda")[:, :100])
    other = kv.DevicePool(0, 1, 4, 16, 256, 64, True)
    with pytest.raises(kv.KVCudaError) as e:
        ws.attn_mass(other, 0, q, lse, *args, mass)
    assert e.value.name == "Unsupported"
    shifted = torch.zeros(2 * 20 * W + 1, device="cuda")[1:].view(2, 1, 20, W)
    with pytest.raises(kv.KVCudaError):  # q not 16-byte aligned
        ws.attn_mass(cache.pool, 0, shifted, lse, *args, mass)
    with pytest.raises(ValueError):  # queries of another width than the rows
        ws.attn_mass(cache.pool, 0, q[..., :512].contiguous(), lse, *args, mass)
    with pytest.raises(ValueError):
        ws.attn_mass(cache.pool, 0, q.half(), lse, *args, mass)
    with pytest.raises(ValueError):
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev.long(), SCALE, mass)
    ws.plan_layers(cache.pool, cache.lens_dev, 2)
    with pytest.raises(kv.KVCudaError):  # a layered plan
        ws.attn_mass(cache.pool, 0, q, lse, *args, mass)


@pytest.mark.parametrize("n_q,heads,bs", [(8, 8, 64), (3, 32, 16), (20, 10, 48), (48, 32, 128), (5, 20, 256)])
def test_many_columns(kv, n_q, heads, bs):
    """Windows of 64 and more columns, from one chunk to eight; 48 x 32 columns of eight entries take
    several passes over the queries.  Sums of old positions decay once."""
    import torch

    lens = [n_q, 127, 128, 129, 255, 1, 2500, 640]
    cache = Paged(kv, lens, bs, True, layers=2, seed=n_q)
    n = len(lens)
    q, lse = queries(cache, range(n), n_q, heads, 3, layer=1)
    mass = torch.rand(n, max(lens) + 3, device="cuda")
    before = mass.clone()
    old = [max(0, x - n_q) for x in lens]
    want, tol = want_mass(cache, range(n), q, lse, mass, 0.9, old, layer=1)
    ws = kv.DecodeWorkspace(0, n, heads)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 1, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, decay=0.9,
                 old_lens=torch.tensor(old, dtype=torch.int32, device="cuda"))
    assert cache.pool.status() == 0
    check(mass, want, tol)
    for b, length in enumerate(lens):
        assert torch.equal(mass[b, length:], before[b, length:])


def test_many_columns_with_uneven_scales(kv):
    """Blocks of a row whose scales span the f16 range, zeros among them, and a bad block."""
    import torch

    from pooldata import arrays

    cache = Paged(kv, [300, 900], 32, True, seed=12)
    _, sc = arrays(cache.pool)
    g = torch.Generator(device="cuda").manual_seed(1)
    power = torch.randint(-12, 1, sc.shape, generator=g, device="cuda").float()
    sc.copy_((sc.float() * 2.0 ** power).half())
    sc[::5, 3] = 0
    sc[7::31] = 0
    n_q, heads = 6, 20
    q, lse = queries(cache, range(2), n_q, heads, 5)
    mass = torch.rand(2, 900, device="cuda")
    before = mass.clone()
    want, tol = want_mass(cache, range(2), q, lse, mass, 1.0, cache.lens)
    tables = cache.tables.clone()
    tables[2] = -1  # positions 64..95 of the first sequence
    ws = kv.DecodeWorkspace(0, 2, heads)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, tables, cache.lens_dev, SCALE, mass)
    assert cache.pool.status() == 0x2
    assert torch.equal(mass[0, 64:96], before[0, 64:96])
    mass[0, 64:96] = want[0, 64:96].float()
    check(mass, want, tol)


def test_many_columns_withheld_and_again(kv):
    import torch

    cache = Paged(kv, [30000, 10000], 64, True, seed=13)
    n_q, heads = 4, 20
    q, lse = queries(cache, range(2), n_q, heads, 5)
    ws = kv.DecodeWorkspace(0, 2, heads)
    ws.plan(cache.pool, cache.lens_dev)
    new = torch.zeros(2, dtype=torch.int32, device="cuda")

    def run():
        m = torch.zeros(2, 30000, device="cuda")
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, m, old_lens=new)
        torch.cuda.synchronize()
        return m

    want = run()
    assert cache.pool.status() == 0
    ws.set_wait_limit(1 << 22)
    for tile in (0, 1):
        ws.test_withhold(tile)
        run()
        assert cache.pool.status() & 0x10
    ws.test_withhold(0xFFFFFFFF)
    ws.set_wait_limit(0)
    assert torch.equal(run(), want) and cache.pool.status() == 0


@pytest.mark.parametrize("n_q", [1, 4])
def test_nan_rows_and_queries_without_positions(kv, n_q):
    """Queries with lse = -inf add nothing, also to rows of NaN and infinities; a live query's NaN shows
    in the rows that have them and in no other."""
    import torch

    from pooldata import arrays

    cache = Paged(kv, [300, 1000], 64, True, seed=14)
    q, lse = queries(cache, range(2), n_q, 20, 6)
    _, sc = arrays(cache.pool)
    for s, value in ((0, float("nan")), (1, float("inf"))):
        sc[torch.from_numpy(cache.rows_at(s, [3, 130])).cuda()] = value
    lse[0] = -math.inf
    mass = torch.rand(2, 1000, device="cuda")
    before = mass.clone()
    ws = kv.DecodeWorkspace(0, 2, 20)
    ws.plan(cache.pool, cache.lens_dev)
    ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, decay=0.5)
    assert torch.equal(mass[0, :300], before[0, :300] * 0.5) and torch.equal(mass[0, 300:], before[0, 300:])
    fine = torch.ones(1000, dtype=torch.bool, device="cuda")
    fine[[3, 130]] = False
    assert torch.isfinite(mass[1, fine]).all() and not torch.isfinite(mass[1, ~fine]).any()


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("tile", [0, 1])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(kv, quant, tile):
    """Units that are never copied: the waits on them end, the status says so, and the same workspace
    gives the same bits as before."""
    import torch

    cache = Paged(kv, [60000, 3000, 20000, 700], 64, quant, seed=11)  # more than two tiles to a CTA
    q, lse = queries(cache, range(4), 1, 20, 6)
    ws = kv.DecodeWorkspace(0, 4, 20)
    ws.plan(cache.pool, cache.lens_dev)
    new = torch.zeros(4, dtype=torch.int32, device="cuda")

    def run():
        m = torch.zeros(4, 60000, device="cuda")
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, m, old_lens=new)
        torch.cuda.synchronize()
        return m

    want = run()
    assert cache.pool.status() == 0
    ws.set_wait_limit(1 << 22)  # about 2 ms
    ws.test_withhold(tile)
    run()
    assert cache.pool.status() & 0x10
    ws.test_withhold(0xFFFFFFFF)
    ws.set_wait_limit(0)
    assert torch.equal(run(), want) and cache.pool.status() == 0


def test_many_columns_between_decodes_and_in_a_graph(kv):
    """The decodes' partials lend their room: a decode after the sums gives the bits of one before, and
    a captured window the bits of an eager one."""
    import torch

    cache = Paged(kv, [5000, 300, 64, 2049], 64, True, seed=15)
    n_q, heads = 16, 20
    q, lse = queries(cache, range(4), n_q, heads, 6)
    ws = kv.DecodeWorkspace(0, 4, heads)
    ws.plan(cache.pool, cache.lens_dev)
    qd = q[:, 0].contiguous()
    outs = [torch.empty(4, heads, 512, device="cuda") for _ in range(4)]
    masses = [torch.zeros(4, 5000, device="cuda") for _ in range(4)]
    decode = lambda o, **k: ws.decode(cache.pool, 0, qd, cache.toff, cache.tables, cache.lens_dev, SCALE, o, **k)
    window = lambda m, **k: ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, m, **k)
    decode(outs[0])
    torch.cuda.synchronize()
    for i in (1, 2):
        window(masses[i])
        decode(outs[i])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream()
        decode(outs[3], stream=s)
        window(masses[3], stream=s)
        decode(outs[3], stream=s)
    for i in range(2):
        masses[3].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(masses[3], masses[1]) and torch.equal(outs[3], outs[0])
    assert torch.equal(masses[1], masses[2]) and torch.equal(outs[1], outs[0]) and torch.equal(outs[2], outs[0])
    assert cache.pool.status() == 0
