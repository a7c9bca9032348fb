"""Limits so short that waits for ordinary loads may run out (a try of the hardware's
barriers may itself take longer than the limit, so they need not): whichever role gives
up first, the call ends, what it had in flight has landed, and the next call is right."""
import pytest

from pooldata import Paged
from test_gpu_mass import SCALE, kv, queries  # noqa: F401 (kv is the module's fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,n_q", [(True, 1), (False, 1), (True, 4)])
def test_waits_that_run_out_at_any_place(kv, quant, n_q):
    import torch

    cache = Paged(kv, [30000, 10000, 300], 64, quant, seed=12)
    q, lse = queries(cache, range(3), n_q, 20, 6)
    ws = kv.DecodeWorkspace(0, 3, 20)
    ws.plan(cache.pool, cache.lens_dev)
    new = torch.zeros(3, dtype=torch.int32, device="cuda")

    def run():
        m = torch.zeros(3, 30000, device="cuda")
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, m, old_lens=new)
        return m

    want = run()
    assert cache.pool.status() == 0
    for limit in (1, 300, 1000, 3000, 10000, 30000):
        ws.set_wait_limit(limit)
        for _ in range(3):
            run()
        assert cache.pool.status() in (0, 0x10)
        ws.set_wait_limit(0)
        assert torch.equal(run(), want) and cache.pool.status() == 0
