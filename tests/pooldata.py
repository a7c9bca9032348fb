"""Helpers of the bounded-cache tests: a DevicePool's memory as torch tensors and
a paged cache of ragged sequences with seeded rows, read back in 64 bits."""
from __future__ import annotations

import numpy as np

R, P, W, BLOCKS = 512, 64, 576, 18


class _Memory:
    def __init__(self, pool, address, shape, kind):
        self.pool = pool  # the tensor keeps the pool alive
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (address, False), "version": 3}


def arrays(pool):
    """The pool's two arrays [rows][...]: (payload int8, scales f16) or (latent f32, rope f32)."""
    import torch

    d = pool.describe()
    rows = d.n_layers * d.num_blocks * d.block_size
    if d.quantized:
        parts = ((d.qs, (rows, d.nblk * 32), "|i1"), (d.sc, (rows, d.nblk), "<f2"))
    else:
        parts = ((d.kv, (rows, d.kv_rank), "<f4"), (d.pe, (rows, d.rope_dim), "<f4"))
    return [torch.as_tensor(_Memory(pool, *x), device=torch.device("cuda", d.device)) for x in parts]


class Paged:
    """Sequences of the given lengths (of `seqs` ids, others empty) over shuffled blocks."""

    def __init__(self, kv, lens, bs, quant, layers=1, seed=1, spare=3, dims=(R, P)):
        import torch

        rng = np.random.default_rng(seed)
        self.lens = [int(x) for x in lens]
        need = [-(-x // bs) for x in self.lens]
        self.nb, self.bs, self.layers = sum(need) + spare, bs, layers
        self.pool = kv.DevicePool(0, layers, self.nb, bs, dims[0], dims[1], quant)
        order = rng.permutation(self.nb).astype(np.int32)
        offs = np.concatenate([[0], np.cumsum(need)]).astype(np.int32)
        self.table = [order[offs[i]:offs[i + 1]].astype(np.int64) for i in range(len(need))]
        self.free = order[offs[-1]:]
        self.toff = torch.from_numpy(offs).cuda()
        self.tables = torch.from_numpy(order[:max(1, offs[-1])].copy()).cuda()
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(seed)
        a, b = arrays(self.pool)
        if quant:
            a.copy_(torch.randint(-127, 128, a.shape, generator=g, device="cuda", dtype=torch.int8))
            b.copy_((torch.rand(b.shape, generator=g, device="cuda") * 0.02 + 0.005).to(torch.float16))
        else:
            a.copy_(torch.randn(a.shape, generator=g, device="cuda"))
            b.copy_(torch.randn(b.shape, generator=g, device="cuda"))

    def rows_at(self, s, positions, layer=0):
        """Physical row indices of positions (numpy int64) of sequence s."""
        p = np.asarray(positions, np.int64)
        return (layer * self.nb + self.table[s][p // self.bs]) * self.bs + p % self.bs

    def values(self, s, layer=0):
        """The cached rows of sequence s as float64 [len][W]."""
        import torch

        at = torch.from_numpy(self.rows_at(s, np.arange(self.lens[s]), layer)).cuda()
        a, b = arrays(self.pool)
        if self.pool.describe().quantized:
            q = a[at].double().view(len(at), a.shape[1] // 32, 32) * b[at].double()[..., None]
            return q.view(len(at), a.shape[1])
        return torch.cat([a[at], b[at]], 1).double()
