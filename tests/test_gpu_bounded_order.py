"""What follows an eviction on another stream runs after its moves.

The eviction's stream is held up by an ordinary kernel, so that its moves are still to
come when the other call is made; nothing is synchronised in between.  Moved rows are
compared byte for byte with the choice that the sums make."""
import gc

import numpy as np
import pytest

from kvdata import SCALE, W
from test_gpu_bounded import BS, P, Step, kv, make  # noqa: F401 (kv is the module's fixture)
from test_gpu_evict import want_keep

pytestmark = pytest.mark.gpu

HOLD = 200_000_000  # clocks, about a tenth of a second
LAYERS = 2


class Evicted:
    """Sequence 0 brought from 1,280 rows to 640 on a held-up side stream: all kept rows come from
    blocks behind the budget, which the host has given back already.  Sequence 1 holds 70 rows,
    the first 64 of them shared with sequence 2."""

    def __init__(self, kv, quant, before=lambda cache: None):
        import torch

        self.c = c = make(kv, [1280, 70, 0], quant, LAYERS, spare=2)
        self.tokens = np.random.default_rng(3).integers(0, 50000, 64).astype(np.uint32)
        prefix = kv.NO_HASH
        for bi in range(4):
            part = self.tokens[bi * BS:(bi + 1) * BS]
            c.seq_cache_block(1, bi, part, prefix)
            prefix = kv.KVCache.computeHash(part, prefix)
        c.seq_reuse_prefix_blocks(2, self.tokens, 4)
        self.rows = [[c.gather(layer, s) for s in range(3)] for layer in range(LAYERS)]
        before(c)
        self.mass = torch.arange(1280, device="cuda", dtype=torch.float32).repeat(LAYERS, 1, 1)
        self.keep = torch.empty(LAYERS, 1, 640, dtype=torch.int32, device="cuda")
        # once within the budget, which changes nothing: kernels loaded and scratch there, so that the host does not wait
        c.evict_dev([1], 640, torch.zeros(LAYERS, 1, 70, device="cuda"), keep_dev=self.keep)
        self.other = torch.cuda.Stream()
        side = torch.cuda.Stream()
        gc.collect()  # an earlier test's cache, freed in between, would wait for the device
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(HOLD)
        c.evict_dev([0], 640, self.mass, 0, 0, keep_dev=self.keep, stream=side)
        assert c.seq_len(0) == 640 and not side.query()

    def check(self, second):
        """Sequences 0 and 1, and 2, whose rows in each layer are to be second(layer)."""
        import torch

        torch.cuda.synchronize()
        assert self.c.pool().status() == 0
        for layer in range(LAYERS):
            assert np.array_equal(self.c.gather(layer, 0), self.rows[layer][0][640:])
            assert np.array_equal(self.c.gather(layer, 1), self.rows[layer][1])
            assert np.array_equal(self.c.gather(layer, 2), second(layer))
        assert np.array_equal(self.mass[:, 0, :640].cpu().numpy(),
                              np.broadcast_to(np.arange(640, 1280, dtype=np.float32), (LAYERS, 640)))


@pytest.mark.parametrize("quant", [True, False])
def test_a_second_eviction_copies_shared_blocks_after_the_first(kv, quant):
    import torch

    e = Evicted(kv, quant)
    mass = torch.rand(LAYERS, 1, 64, generator=torch.Generator().manual_seed(1)).cuda()
    m = mass.cpu().numpy()
    e.other.wait_stream(torch.cuda.current_stream())
    e.c.evict_dev([2], 40, mass, 4, 8, stream=e.other)
    assert len(set(e.c.seq_block_table(2)) & set(e.c.seq_block_table(1))) == 0
    e.check(lambda layer: e.rows[layer][2][want_keep(m[layer, 0], 64, 40, 4, 8)])


@pytest.mark.parametrize("quant", [True, False])
def test_appends_into_shared_blocks_after_an_eviction(kv, quant):
    import torch

    e = Evicted(kv, quant)
    c = e.c
    rows = np.random.default_rng(9).standard_normal((LAYERS, 1, W)).astype(np.float32)
    dev = torch.from_numpy(rows).cuda()
    ids, pos = np.array([2], np.uint32), np.array([60], np.uint32)
    ids_dev, pos_dev = torch.tensor([2], dtype=torch.int32).cuda(), torch.tensor([60], dtype=torch.int32).cuda()
    e.other.wait_stream(torch.cuda.current_stream())
    c.seq_truncate(2, 60)
    c.seq_ensure_capacity(2, 61)
    for layer in range(LAYERS):
        c.appendBatch_dev(layer, ids, pos, ids_dev, pos_dev, dev[layer], stream=e.other)
    torch.cuda.synchronize()
    want = [c.gather(layer, 2) for layer in range(LAYERS)]
    for layer in range(LAYERS):
        assert np.array_equal(want[layer][:60], e.rows[layer][2][:60])
        assert np.abs(want[layer][60] - rows[layer, 0]).max() <= (0.023 if quant else 0)  # values below 5: half a step, and the scale in f16
    e.check(lambda layer: want[layer])


def test_host_appends_and_steps_after_an_eviction(kv):
    import torch

    e = Evicted(kv, True)
    c = e.c
    rows = np.random.default_rng(9).standard_normal((1, W)).astype(np.float32)
    c.seq_truncate(2, 60)
    c.seq_ensure_capacity(2, 61)
    for layer in range(LAYERS):  # on the cache's own stream
        c.appendBatch(layer, np.array([2], np.uint32), np.array([60], np.uint32), rows)
    e.check(lambda layer: np.concatenate([e.rows[layer][2][:60], c.gather(layer, 2)[60:]]))
    f = Evicted(kv, True)
    c = f.c
    st = Step(1, 2)
    f.other.wait_stream(torch.cuda.current_stream())
    c.seq_truncate(2, 60)
    c.seq_ensure_capacity(2, 61)
    for layer in range(LAYERS):
        st.run(c, layer, [2], [60], kv.Rope(P), stream=f.other)
    f.check(lambda layer: np.concatenate([f.rows[layer][2][:60], c.gather(layer, 2)[60:]]))


@pytest.mark.parametrize("how", ["v1", "v2", "background"])
def test_a_save_after_an_eviction_holds_its_rows(kv, tmp_path, how):
    e = Evicted(kv, True)
    at = tmp_path / "save.ckpt"
    if how == "v1":  # sequence 0 alone
        e.c.saveToFile(at)
    elif how == "v2":
        e.c.saveToFileV2(at)
    else:
        e.c.saveToFileV2Async(at).wait()
    e.check(lambda layer: e.rows[layer][2])
    d = kv.KVCache.with_blocks(LAYERS, 512, P, e.c.num_blocks, BS, quantized=True)
    if how == "v1":
        d.loadFromFile(at)
    else:
        d.loadFromFileV2(at)
    for layer in range(LAYERS):
        assert np.array_equal(d.gather(layer, 0), e.rows[layer][0][640:])
        for s in (1, 2) if how != "v1" else ():
            assert np.array_equal(d.gather(layer, s), e.rows[layer][s])


def test_a_load_after_an_eviction_keeps_what_it_read(kv, tmp_path):
    e = Evicted(kv, True, before=lambda cache: cache.saveToFileV2(tmp_path / "save.ckpt"))
    e.c.loadFromFileV2(tmp_path / "save.ckpt")
    for layer in range(LAYERS):
        for s in range(3):
            assert np.array_equal(e.c.gather(layer, s), e.rows[layer][s])
