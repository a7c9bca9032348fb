"""What kvcu_attn_mass reports of entries that it cannot read, by both of its kernels."""
import pytest

from pooldata import Paged
from test_gpu_mass import SCALE, check, kv, queries, want_mass  # noqa: F401 (kv is the module's fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,n_q", [(True, 1), (False, 1), (False, 3), (True, 3)])
def test_a_sequence_that_is_not_there_is_reported(kv, quant, n_q):
    """It has no tokens, but the plan lists it: its sums stay, and the other entry's are right."""
    import torch

    cache = Paged(kv, [200, 300], 16, quant, seed=5)
    q, lse = queries(cache, [1, 0], n_q, 20, 4)
    mass = torch.rand(2, 300, device="cuda")
    before = mass.clone()
    for bad in (2, 7, -1):
        ids = torch.tensor([1, bad], dtype=torch.int32, device="cuda")
        ws = kv.DecodeWorkspace(0, 2, 20)
        ws.plan(cache.pool, cache.lens_dev, seq_ids=ids)
        mass.copy_(before)
        ws.attn_mass(cache.pool, 0, q, lse, cache.toff, cache.tables, cache.lens_dev, SCALE, mass, seq_ids=ids)
        assert cache.pool.status() == 0x4
        assert torch.equal(mass[1], before[1])
        want, tol = want_mass(cache, [1], q[:1], lse[:1], before[:1], 1.0, [300])
        check(mass[:1], want, tol)
