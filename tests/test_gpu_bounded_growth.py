"""The launches of the weights: sequences that grew between a step and the call, windows of queries."""
import numpy as np
import pytest

from kvdata import SCALE, W
from test_gpu_bounded import Cached, P, Step, kv, make  # noqa: F401 (kv is the module's fixture)
from test_gpu_mass import check, want_mass

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grown,launches", [(0, 1), (7, 1), (900, 2)])
def test_the_steps_plan_serves_while_the_batch_grew_little(kv, grown, launches):
    import torch

    lens = [40, 20]
    c = make(kv, lens, True, 1, spare=100)
    st = Step(2, 6)
    c.seq_ensure_capacity(0, 64), c.seq_ensure_capacity(1, 1000)
    st.run(c, 0, [0, 1], lens, kv.Rope(P))
    lens = [41, 21 + grown]
    if grown:
        rows = np.random.default_rng(4).standard_normal((grown, W)).astype(np.float32)
        c.appendBatch(0, np.full(grown, 1, np.uint32), np.arange(21, 21 + grown, dtype=np.uint32), rows)
    q, lse = torch.randn(2, 20, W, device="cuda") * 0.05, torch.empty(2, 20, device="cuda")
    view = Cached(c, lens)
    for s in range(2):
        lse[s] = torch.logsumexp(q[s].double() @ view.values(s).T * SCALE, 1).float()
    mass = torch.ones(2, 1000, device="cuda")
    want, tol = want_mass(view, [0, 1], q[:, None], lse[:, None], mass, 0.5, lens)
    c.attnMass_dev(0, [0, 1], q, lse, SCALE, mass, decay=0.5)
    assert c.last_launches == launches
    assert c.pool().status() == 0
    check(mass, want, tol)


@pytest.mark.parametrize("quant,n_q,launches", [(True, 1, 1), (True, 2, 1), (True, 3, 2), (True, 40, 2), (False, 40, 1)])
def test_launches_of_a_window(kv, quant, n_q, launches):
    """Many columns of Q8_0 rows are laid out first; a plan, where the batch is another one, comes on top."""
    import torch

    c = make(kv, [300], quant, 1)
    q = torch.randn(1, n_q, 20, W, device="cuda") * 0.05
    mass, lse = torch.zeros(1, 300, device="cuda"), torch.zeros(1, n_q, 20, device="cuda")
    for plan in (1, 0):
        c.attnMass_dev(0, [0], q, lse, SCALE, mass)
        assert c.last_launches == launches + plan
