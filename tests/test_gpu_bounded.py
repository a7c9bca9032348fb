"""A cache that stays within a budget: the MLA step with rotary positions of its own,
the weights the cached positions receive, the eviction, and steps after it, each
stage against 64 bits on the stage's own inputs.

Tolerances.  Moved rows, their sums and untouched rows are equal in every bit.  The
row a step appends is RMSNorm and a rotation in f32: a few roundings of its largest
value, plus half a Q8_0 step and the f16 rounding of its scale where quantised.  The
weights' bound is test_gpu_mass's; the decode's log-sum-exp and the step's output
carry the project's attention tolerance."""
import math

import numpy as np
import pytest

from kvdata import REL_TOL, SCALE, W, rel_err_rows
from test_gpu_evict import want_keep
from test_gpu_mass import check, want_mass

pytestmark = pytest.mark.gpu

R, P, BS = 512, 64, 16
H, QK_NOPE, V_DIM, EPS = 20, 128, 128, 1e-6


@pytest.fixture(scope="module")
def kv():
    import torch

    import kvcu

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    kvcu.init(0)
    return kvcu


def make(kv, lens, quant, layers=2, seed=5, spare=24, bs=BS):
    nb = sum(-(-x // bs) for x in lens) + spare
    c = kv.KVCache.with_blocks(layers, R, P, nb, bs, quantized=quant)
    for _ in range(len(lens) - 1):
        c.seq_create()
    rng = np.random.default_rng(seed)
    for s, length in enumerate(lens):
        c.seq_ensure_capacity(s, max(length, 1))
        for layer in range(layers):
            if length:
                c.appendBatch(layer, np.full(length, s, np.uint32), np.arange(length, dtype=np.uint32),
                              rng.standard_normal((length, W)).astype(np.float32))
    return c


class Cached:
    """The cache as want_mass reads it."""

    def __init__(self, c, lens):
        self.c, self.lens = c, lens

    def values(self, s, layer=0):
        import torch

        return torch.from_numpy(self.c.gather(layer, s)).cuda().double()


def rotated(x, pos, freq):
    """Interleaved pairs of x [..., P] (64 bits) turned by pos * freq."""
    a = pos * freq
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(a) - x[..., 1::2] * np.sin(a)
    out[..., 1::2] = x[..., 0::2] * np.sin(a) + x[..., 1::2] * np.cos(a)
    return out


class Step:
    """One layer's weights and random activations."""

    def __init__(self, n, seed):
        import torch

        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.q, self.kv_a, self.w = r(n, H, QK_NOPE + P), r(n, R + P), 1 + 0.1 * r(R)
        self.k_b, self.v_b = r(H * QK_NOPE, R) / math.sqrt(R), r(H * V_DIM, R) / math.sqrt(R)
        nan = lambda *s: torch.full(s, float("nan"), device="cuda")
        self.attn, self.q_abs, self.lse = nan(n, H, V_DIM), nan(n, H, W), nan(n, H)

    def run(self, c, layer, ids, pos, rope, rope_pos=None, outputs=True, stream=None):
        c.mla_step_rope_dev(layer, ids, pos, rope, self.q, self.kv_a, self.w, EPS, self.k_b, self.v_b, QK_NOPE, V_DIM,
                            SCALE, self.attn, rope_positions=rope_pos, q_abs=self.q_abs if outputs else None,
                            lse=self.lse if outputs else None, stream=stream)

    def check(self, c, layer, ids, pos, rope_pos, freq, quant, mag=1.0):
        """The appended rows, absorbed queries, log-sum-exp and output against 64 bits."""
        d = lambda t: t.cpu().numpy().astype(np.float64)
        q, kv_a, k_b, v_b = d(self.q), d(self.kv_a), d(self.k_b).reshape(H, QK_NOPE, R), d(self.v_b).reshape(H, V_DIM, R)
        q_abs, lse, attn = d(self.q_abs), d(self.lse), d(self.attn)
        want_out = np.empty_like(attn)
        for b, s in enumerate(ids):
            x = kv_a[b, :R]
            row = np.concatenate([x / np.sqrt((x * x).mean() + EPS) * d(self.w),
                                  mag * rotated(kv_a[b, R:], rope_pos[b], freq)])
            rows = c.gather(layer, s).astype(np.float64)
            amax = np.repeat(np.abs(row).reshape(-1, 32).max(1), 32)
            step = amax / 127 * 0.5 + np.abs(row) * 2.0 ** -11 if quant else 0.0
            assert (np.abs(rows[pos[b]] - row) <= step * 1.001 + 32 * 2.0 ** -24 * np.abs(row).max()).all()
            qr = mag * rotated(q[b, :, QK_NOPE:], rope_pos[b], freq)
            assert np.abs(q_abs[b, :, R:] - qr).max() <= 8 * 2.0 ** -24 * np.abs(qr).max()
            qa = np.einsum("hk,hkr->hr", q[b, :, :QK_NOPE], k_b)
            assert rel_err_rows(q_abs[b, :, :R], qa) <= REL_TOL
            # the newest token's latent takes part as it was before its rounding to the cache
            keys = rows.copy()
            keys[pos[b], :R] = row[:R]
            sc = q_abs[b] @ keys.T * SCALE
            top = sc.max(1, keepdims=True)
            e = np.exp(sc - top)
            assert np.abs(lse[b] - (top[:, 0] + np.log(e.sum(1)))).max() <= REL_TOL
            want_out[b] = np.einsum("hr,hvr->hv", e / e.sum(1, keepdims=True) @ keys[:, :R], v_b)
        assert np.isfinite(attn).all()
        assert rel_err_rows(attn, want_out) <= REL_TOL


@pytest.mark.parametrize("quant", [True, False])
def test_steps_with_evictions_between(kv, quant):
    import torch

    layers, budget, sink, recent, slack = 2, 96, 4, 24, 3
    lens = [0, 40, 93, 150]
    n = len(lens)
    c = make(kv, lens, quant, layers)
    rope = kv.Rope(P, base=50000.0, scaling="yarn", factor=4.0, orig_ctx=64)
    freq, mag = rope.frequencies()
    ids, tokens = list(range(n)), list(lens)
    mass = torch.zeros(layers, n, 160, device="cuda")
    evictions = 0
    for step in range(8):
        for s in ids:
            c.seq_ensure_capacity(s, lens[s] + 1)
        old = np.array(lens, np.uint32)
        for layer in range(layers):
            st = Step(n, 100 * step + layer)
            st.run(c, layer, ids, lens, rope, tokens)
            before = mass[layer].clone()
            c.attnMass_dev(layer, ids, st.q_abs, st.lse, SCALE, mass[layer], decay=0.97, old_lens=old)
            assert c.last_launches == 1  # on the step's plan
            torch.cuda.synchronize()
            assert c.pool().status() == 0
            now = [x + 1 for x in lens]
            st.check(c, layer, ids, lens, tokens, freq, quant, mag)
            want, tol = want_mass(Cached(c, now), ids, st.q_abs[:, None], st.lse[:, None], before, 0.97, old, layer=layer)
            check(mass[layer], want, tol)
        lens = [x + 1 for x in lens]
        tokens = [x + 1 for x in tokens]
        if max(lens) < budget + slack:
            continue
        evictions += 1
        rows = [[c.gather(layer, s) for s in ids] for layer in range(layers)]
        m = mass.cpu().numpy()
        keep = torch.full((layers, n, budget), 7, dtype=torch.int32, device="cuda")
        free = c.numFreeBlocks()
        held = [len(c.seq_block_table(s)) for s in ids]
        c.evict_dev(ids, budget, mass, sink, recent, keep_dev=keep)
        torch.cuda.synchronize()
        assert c.pool().status() == 0
        k, after = keep.cpu().numpy(), mass.cpu().numpy()
        for s in ids:
            left = min(lens[s], budget)
            assert c.seq_len(s) == left
            for layer in range(layers):
                want = want_keep(m[layer, s], lens[s], budget, sink, recent)
                assert np.array_equal(k[layer, s, :left], want) and (k[layer, s, left:] == -1).all()
                assert np.array_equal(c.gather(layer, s), rows[layer][s][want])
                assert np.array_equal(after[layer, s, :left], m[layer, s, want])
        assert c.numFreeBlocks() - free == sum(h - len(c.seq_block_table(s)) for h, s in zip(held, ids))
        lens = [min(x, budget) for x in lens]
    assert evictions >= 2
    live = [b for s in ids for b in c.seq_block_table(s)]
    assert len(set(live)) == len(live) and c.numFreeBlocks() + len(live) == c.num_blocks


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk"])
def test_step_at_its_own_rotary_positions(kv, quant, scaling):
    import torch

    lens, at = [0, 1, 63, 64, 300], [0, 9, 5000, 64, 131071]
    c = make(kv, lens, quant, 1)
    for s, x in enumerate(lens):
        c.seq_ensure_capacity(s, x + 1)
    rope = kv.Rope(P, base=10000.0, scaling=scaling, factor=1.0 if scaling == "none" else 8.0, orig_ctx=4096)
    freq, mag = rope.frequencies()
    assert mag == 1.0
    st = Step(len(lens), 3)
    st.run(c, 0, range(len(lens)), lens, rope, at)
    torch.cuda.synchronize()
    assert c.pool().status() == 0
    st.check(c, 0, range(len(lens)), lens, at, freq, quant)


def test_step_without_positions_is_the_plain_step(kv):
    """The cache positions are the default, and the outputs may be left out."""
    import torch

    lens = [0, 5, 64, 130]
    ids = range(len(lens))
    a, b = make(kv, lens, True, 1), make(kv, lens, True, 1)
    for s, x in enumerate(lens):
        a.seq_ensure_capacity(s, x + 1), b.seq_ensure_capacity(s, x + 1)
    st, plain = Step(4, 8), Step(4, 8)
    with_out = Step(4, 8)
    st.run(a, 0, ids, lens, kv.Rope(P), outputs=False)
    b.mla_step_dev(0, ids, lens, plain.q, plain.kv_a, plain.w, EPS, 10000.0, plain.k_b, plain.v_b, QK_NOPE, V_DIM, SCALE,
                   plain.attn)
    assert rel_err_rows(st.attn.cpu().numpy(), plain.attn.cpu().numpy()) <= 2 * REL_TOL  # each within REL_TOL
    # again over the same positions, with the outputs: the same bits
    for s, x in enumerate(lens):
        a.seq_truncate(s, x)
        a.seq_ensure_capacity(s, x + 1)
    with_out.run(a, 0, ids, lens, kv.Rope(P))
    assert torch.equal(with_out.attn, st.attn) and torch.isfinite(with_out.lse).all()


@pytest.mark.parametrize("quant", [True, False])
def test_decode_and_prompt_window_give_their_log_sum_exp(kv, quant):
    import torch

    lens = [77, 1, 900]
    c = make(kv, lens, quant, 2, bs=64)
    q = torch.randn(3, H, W, device="cuda") * 0.05
    out, ref, lse = torch.empty(3, H, R, device="cuda"), torch.empty(3, H, R, device="cuda"), torch.empty(3, H,
                                                                                                         device="cuda")
    c.mlaDecode_dev(1, [0, 1, 2], q, SCALE, ref)
    c.mlaDecodeLse_dev(1, [0, 1, 2], q, SCALE, out, lse)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)
    view = Cached(c, lens)
    for s in range(3):
        want = torch.logsumexp(q[s].double() @ view.values(s, 1).T * SCALE, 1)
        assert (lse[s].double() - want).abs().max() <= REL_TOL
    mass = torch.zeros(3, 1000, device="cuda")
    c.attnMass_dev(1, [0, 1, 2], q, lse, SCALE, mass)
    want, tol = want_mass(view, [0, 1, 2], q[:, None], lse[:, None], torch.zeros_like(mass), 1.0, lens, layer=1)
    check(mass, want, tol)
    # a prompt's last positions: one sequence, a window of queries
    n_q = 13
    qp = torch.randn(n_q, H, W, device="cuda") * 0.05
    o1, o2, lp = torch.empty(n_q, H, R, device="cuda"), torch.empty(n_q, H, R, device="cuda"), torch.empty(
        1, n_q, H, device="cuda")
    c.mlaAttentionBatch_dev(0, 2, 900 - n_q, qp, SCALE, o1)
    c.mlaAttentionBatchLse_dev(0, 2, 900 - n_q, qp, SCALE, o2, lp)
    assert torch.equal(o1, o2)
    mass = torch.full((1, 1000), 3.0, device="cuda")
    c.attnMass_dev(0, [2], qp[None], lp, SCALE, mass, old_lens=[0])
    want, tol = want_mass(view, [2], qp[None], lp, torch.full_like(mass, 3.0), 1.0, [0])
    check(mass, want, tol)
    assert abs(float(mass[0, :900].sum()) / (n_q * H) - 1) <= REL_TOL


def test_weights_on_the_plan_of_another_batch(kv):
    """After a step of other sequences, a refused step, or an eviction, the sums are of the sequences asked for."""
    import torch

    lens = [30, 200, 64, 120]
    c = make(kv, lens, True, 1)
    for s, x in enumerate(lens):
        c.seq_ensure_capacity(s, x + 1)
    rope = kv.Rope(P)
    st = Step(2, 4)
    st.run(c, 0, [0, 1], lens[:2], rope)
    with pytest.raises(kv.KVCudaError):  # refused after its batch was looked at
        c.mla_step_rope_dev(0, [2, 3], lens[2:], rope, st.q, st.kv_a, st.w, EPS, st.k_b, st.v_b, 0, V_DIM, SCALE, st.attn)
    lens = [31, 201, 64, 120]
    q = torch.randn(4, H, W, device="cuda") * 0.05
    out, lse = torch.empty(4, H, R, device="cuda"), torch.empty(4, H, device="cuda")
    mass = torch.zeros(1, 4, 256, device="cuda")
    for ids in ([0, 1], [2, 3], [1, 0], [3, 1, 0, 2]):
        n = len(ids)
        view = Cached(c, lens)
        for b, s in enumerate(ids):
            lse[b] = torch.logsumexp(q[b].double() @ view.values(s).T * SCALE, 1).float()
        m = torch.zeros(n, 256, device="cuda")
        c.attnMass_dev(0, ids, q[:n], lse[:n], SCALE, m)
        want, tol = want_mass(view, ids, q[:n, None], lse[:n, None], torch.zeros_like(m), 1.0, lens)
        check(m, want, tol)
        if ids == [1, 0]:
            mass[0, 0], mass[0, 1] = m[1], m[0]
            c.evict_dev([0, 1, 2, 3], 70, mass, 2, 8)
            lens = [31, 70, 64, 70]


@pytest.mark.parametrize("quant", [True, False])
def test_shared_prefix_blocks_are_copied(kv, quant):
    import torch

    c = make(kv, [74, 0], quant, 2)
    rng = np.random.default_rng(2)
    t0 = rng.integers(0, 50000, 74).astype(np.uint32)
    prefix = kv.NO_HASH
    for bi in range(4):
        c.seq_cache_block(0, bi, t0[bi * BS:(bi + 1) * BS], prefix)
        prefix = kv.KVCache.computeHash(t0[bi * BS:(bi + 1) * BS], prefix)
    c.seq_reuse_prefix_blocks(1, t0, 4)
    assert c.seq_len(1) == 64
    first = [c.gather(layer, 0) for layer in range(2)]
    shared = c.seq_block_table(0)
    mass = torch.rand(2, 1, 64, device="cuda")
    c.evict_dev([1], 40, mass, BS, 4)
    assert c.pool().status() == 0
    assert c.seq_len(1) == 40 and c.seq_block_table(0) == shared
    for layer in range(2):
        assert np.array_equal(c.gather(layer, 0), first[layer])
        assert len(c.gather(layer, 1)) == 40 and np.array_equal(c.gather(layer, 1)[:BS], first[layer][:BS])
        assert (np.abs(c.gather(layer, 1)[:, None] - first[layer][None, :64]).max(2) == 0).any(1).all()
    assert c.seq_block_table(1)[0] == shared[0] and not set(c.seq_block_table(1)[1:]) & set(shared)
    assert c.findPrefixBlocks(t0) == 4  # the first sequence's blocks are what their hash says
    assert [c.refcount(b) for b in shared] == [2, 1, 1, 1, 1]
    # now its own eviction rewrites them: only the untouched first block is a prefix any more
    mass0 = torch.rand(2, 1, 74, device="cuda")
    c.evict_dev([0], 40, mass0, BS, 4)
    assert c.seq_block_table(0) == shared[:3] and c.findPrefixBlocks(t0) == 1


def test_eviction_while_a_save_runs(kv, tmp_path):
    import torch

    lens = [3000, 700, 64]
    c = make(kv, lens, True, 2, spare=300, bs=64)
    torch.cuda.synchronize()
    snap = [[c.gather(layer, s) for s in range(3)] for layer in range(2)]
    job = c.saveToFileV2Async(tmp_path / "save.ckpt")
    mass = torch.rand(2, 3, 3000, device="cuda")
    m = mass.cpu().numpy()
    c.evict_dev([0, 1, 2], 256, mass, 4, 32)
    now = [[c.gather(layer, s) for s in range(3)] for layer in range(2)]
    job.wait()
    d = kv.KVCache.with_blocks(2, R, P, c.num_blocks, 64, quantized=True)
    d.loadFromFileV2(tmp_path / "save.ckpt")
    for s in range(3):
        assert d.seq_len(s) == lens[s] and c.seq_len(s) == min(lens[s], 256)
        for layer in range(2):
            assert np.array_equal(d.gather(layer, s), snap[layer][s])
            assert np.array_equal(now[layer][s], snap[layer][s][want_keep(m[layer, s], lens[s], 256, 4, 32)])
    live = [b for s in range(3) for b in c.seq_block_table(s)]
    assert c.numFreeBlocks() + len(set(live)) == c.num_blocks


def test_on_another_stream(kv):
    """Two evictions one after the other on a side stream share the cache's scratch."""
    import torch

    c = make(kv, [500, 300, 200], True, 2)
    mass = torch.rand(2, 3, 512, device="cuda")
    rows = [[c.gather(layer, s) for s in range(3)] for layer in range(2)]
    m = mass.cpu().numpy()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.evict_dev([0, 1, 2], 250, mass, 4, 32, stream=side)
    with torch.cuda.stream(side):
        left = mass[:, [0, 2]].contiguous()  # of the rows that are left
        again = left.clone()
    c.evict_dev([0, 2], 180, again, 4, 32, stream=side)
    side.synchronize()
    assert c.pool().status() == 0
    lm = left.cpu().numpy()
    for layer in range(2):
        for s, x in enumerate([500, 300, 200]):
            want = rows[layer][s][want_keep(m[layer, s], x, 250, 4, 32)]
            if s != 1:
                want = want[want_keep(lm[layer, s // 2], len(want), 180, 4, 32)]
            assert np.array_equal(c.gather(layer, s), want)


def test_sequences_within_the_budget_stay(kv):
    import torch

    c = make(kv, [50, 0, 64], True, 2)
    rows = [[c.gather(layer, s) for s in range(3)] for layer in range(2)]
    tables = [c.seq_block_table(s) for s in range(3)]
    mass = torch.full((2, 3, 64), float("nan"), device="cuda")
    keep = torch.full((2, 3, 64), 9, dtype=torch.int32, device="cuda")
    c.evict_dev([0, 1, 2], 64, mass, 64, 0)
    assert c.last_launches == 0  # nothing to do
    c.evict_dev([0, 1, 2], 64, mass, 0, 64, keep_dev=keep)
    k = keep.cpu().numpy()
    for s, x in enumerate([50, 0, 64]):
        assert c.seq_len(s) == x and c.seq_block_table(s) == tables[s]
        for layer in range(2):
            assert np.array_equal(c.gather(layer, s), rows[layer][s])
            assert np.array_equal(k[layer, s, :x], np.arange(x)) and (k[layer, s, x:] == -1).all()


def test_refusals(kv):
    import torch

    c = make(kv, [100, 40], True, 1, spare=1)
    mass = torch.rand(1, 2, 128, device="cuda")

    def refused(name, f, *a, **k):
        with pytest.raises(kv.KVCudaError) as e:
            f(*a, **k)
        assert e.value.name == name, e.value.name

    refused("InvalidArgument", c.evict_dev, [0, 2], 64, mass)         # no such sequence
    refused("InvalidArgument", c.evict_dev, [0, 0], 64, mass)         # twice
    refused("InvalidArgument", c.evict_dev, [0, 1], 0, mass)
    refused("InvalidArgument", c.evict_dev, [0, 1], 64, mass, 40, 25)  # more ends than budget
    refused("InvalidArgument", c.evict_dev, [0, 1], 64, mass[:, :, :99].contiguous())  # shorter than a sequence
    with pytest.raises(ValueError):
        c.evict_dev([0, 1], 64, mass[0])
    with pytest.raises(ValueError):
        c.evict_dev([0, 1], 64, mass, keep_dev=torch.zeros(1, 2, 63, dtype=torch.int32, device="cuda"))
    # no block left for the copy of a shared one: nothing moves
    t = np.arange(96, dtype=np.uint32)
    prefix = kv.NO_HASH
    for bi in range(6):
        c.seq_cache_block(0, bi, t[bi * BS:(bi + 1) * BS], prefix)
        prefix = kv.KVCache.computeHash(t[bi * BS:(bi + 1) * BS], prefix)
    s = c.seq_create()
    c.seq_reuse_prefix_blocks(s, t, 6)
    rows, other = c.gather(0, s), c.gather(0, 0)
    refused("OutOfKVCacheBlocks", c.evict_dev, [s], 64, torch.rand(1, 1, 96, device="cuda"))
    assert c.seq_len(s) == 96 and np.array_equal(c.gather(0, s), rows) and np.array_equal(c.gather(0, 0), other)
    q, lse = torch.randn(1, H, W, device="cuda"), torch.zeros(1, H, device="cuda")
    row = torch.zeros(1, 128, device="cuda")
    refused("LayerOutOfBounds", c.attnMass_dev, 1, [0], q, lse, SCALE, row)
    refused("InvalidArgument", c.attnMass_dev, 0, [9], q, lse, SCALE, row)
    refused("InvalidArgument", c.attnMass_dev, 0, [0], q, lse, SCALE, row[:, :99].contiguous())
    with pytest.raises(ValueError):
        c.attnMass_dev(0, [0, 1], q, lse, SCALE, row)
    with pytest.raises(ValueError):
        c.attnMass_dev(0, [0], q, lse[:, :19], SCALE, row)
    with pytest.raises(ValueError):
        c.attnMass_dev(0, [0], q[..., :512].contiguous(), lse, SCALE, row)
    with pytest.raises(ValueError):
        c.mlaDecodeLse_dev(0, [0], q, SCALE, torch.zeros(1, H, R, device="cuda"), lse[:, :19])
    with pytest.raises(ValueError):
        c.evict_dev([0, 1], 64, mass.double())
    st = Step(1, 1)
    refused("InvalidArgument", st.run, c, 0, [1], [40], kv.Rope(32))   # another rotary part than the cache's
    refused("PositionOutOfBounds", st.run, c, 0, [1], [200], kv.Rope(P))
    st.q_abs = torch.zeros(H * W + 1, device="cuda")[1:].view(1, H, W)
    refused("InvalidArgument", st.run, c, 0, [1], [40], kv.Rope(P))    # not 16-byte aligned
    with pytest.raises(ValueError):
        st.run(c, 0, [1], [40], kv.Rope(P), rope_pos=[1, 2])
