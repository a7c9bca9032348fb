"""The measured cases of the operators that keep a long context in a bounded paged MLA cache.

Four operators over the paged cache of 512-wide latents and 64-wide rotary keys:

  mass     the attention weight that every cached position got from a step's queries, added to a running
           sum per position: mass[p] = decay * mass[p] + sum over queries and heads of exp(scale * q . k_p - lse)
  select   which positions stay under a budget: the first `sink`, the last `recent` and, between them,
           those of the largest mass (ties: the lowest position), as an ascending list
  compact  the kept rows of every layer moved to the front of their sequences, in place, through the block
           tables, and their masses with them
  rope     rotary positions of the query heads' rotary part and of the rotary key: interleaved or half layout,
           plain, linear, NTK or by-parts (YaRN) scaled frequencies; its transpose is the gradient

`run` computes them in plain torch operations, or, with `own` set, by the library's calls.
"""
import math
import os
import random
import sys

import torch

own = False

R, P = 512, 64   # latent and rotary width of a cached row
W = R + P
BLOCKS = W // 32  # 32-value blocks of a Q8_0 row
SCALE = 1.0 / math.sqrt(192.0)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _kvcu():
    """The library's Python binding (only where `own` is set)."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mobile-moe.zig_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import kvcu
    return kvcu


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one chat sequence in its first answer: a layer's call is all latency
        {"name": "mass one short", "op": "mass", "n": 1, "lo": 777, "hi": 777, "n_q": 1, "heads": 20, "block": 16,
         "quant": True, "decay": 1.0},
        # a serving batch of ragged contexts, the step's ordinary call
        {"name": "mass batch", "op": "mass", "n": 64, "lo": 128, "hi": 32768, "n_q": 1, "heads": 20, "block": 64,
         "quant": True, "decay": 0.98},
        # the largest batch: the cache's long-context workload, cut to 192 sequences
        {"name": "mass large batch", "op": "mass", "n": 192, "lo": 128, "hi": 65536, "n_q": 1, "heads": 20, "block": 64,
         "quant": True, "decay": 1.0},
        # after a prompt: the last 32 positions' queries say which rows matter
        {"name": "mass prompt window", "op": "mass", "n": 2, "lo": 12289, "hi": 16384, "n_q": 32, "heads": 20,
         "block": 64, "quant": True, "decay": 1.0},
        # a cache that was not quantised
        {"name": "mass f32 rows", "op": "mass", "n": 16, "lo": 1000, "hi": 8191, "n_q": 1, "heads": 20, "block": 16,
         "quant": False, "decay": 1.0},
        # a sequence that has just passed its budget
        {"name": "select one short", "op": "select", "layers": 8, "n": 1, "lo": 641, "hi": 641, "budget": 512, "sink": 4,
         "recent": 64},
        # a batch's contexts brought down to 2k rows each
        {"name": "select batch", "op": "select", "layers": 8, "n": 64, "lo": 1500, "hi": 65536, "budget": 2048,
         "sink": 16, "recent": 256},
        # the rows of that one short sequence
        {"name": "compact one short", "op": "compact", "layers": 8, "n": 1, "lo": 641, "hi": 641, "budget": 512,
         "block": 16, "quant": True},
        # the batch's rows in all layers
        {"name": "compact batch", "op": "compact", "layers": 8, "n": 64, "lo": 1500, "hi": 32768, "budget": 2048,
         "block": 64, "quant": True},
        # one decode step's query heads and rotary key, as the step's f32 path has them
        {"name": "rope one token", "op": "rope", "n": 1, "q_heads": 20, "k_heads": 1, "nope": 128, "rot": 64,
         "layout": "interleaved", "scaling": "none", "dtype": "f32", "transpose": False, "far": 65536},
        # a prompt chunk, half layout, frequencies scaled by parts for a 16 times longer context
        {"name": "rope prompt", "op": "rope", "n": 8191, "q_heads": 20, "k_heads": 1, "nope": 128, "rot": 64,
         "layout": "half", "scaling": "yarn", "dtype": "bf16", "transpose": False, "far": 1048576},
        # the gradient of a batch of rotated heads without an unrotated part
        {"name": "rope gradient", "op": "rope", "n": 4096, "q_heads": 32, "k_heads": 8, "nope": 0, "rot": 128,
         "layout": "interleaved", "scaling": "ntk", "dtype": "f32", "transpose": True, "far": 131072},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["mass", "mass", "select", "compact", "rope"])
    if op == "mass":
        quant, n_q = rng.random() < 0.75, 1
        n, lo, hi = _log(rng, 1, 128), _log(rng, 1, 2048), _log(rng, 2048, 32768)
        if rng.random() < 0.25:
            n_q = _log(rng, 2, 48)
            n, lo, hi = min(n, 4), max(lo, n_q), min(hi, 12000)
        if not quant:
            n, hi = min(n, 16), min(hi, 6000 if n_q > 1 else 8192)
            n_q = min(n_q, 8)
        return {"op": op, "n": n, "lo": min(lo, hi), "hi": hi, "n_q": n_q, "heads": rng.choice([4, 8, 16, 20, 20, 24, 32]),
                "block": rng.choice([16, 32, 64, 128]), "quant": quant, "decay": rng.choice([1.0, 0.9, 0.98])}
    if op == "select":
        budget = _log(rng, 16, 4096)
        lo = max(1, int(budget * rng.uniform(0.5, 1.5)))
        return {"op": op, "layers": rng.randint(1, 8), "n": _log(rng, 1, 64), "lo": lo, "hi": lo + _log(rng, 1, 50000),
                "budget": budget, "sink": rng.randint(0, budget // 4), "recent": rng.randint(0, budget // 2)}
    if op == "compact":
        budget = _log(rng, 16, 2048)
        lo = max(1, int(budget * rng.uniform(0.5, 1.5)))
        quant = rng.random() < 0.7
        return {"op": op, "layers": rng.randint(1, 8), "n": _log(rng, 1, 64 if quant else 16), "lo": lo,
                "hi": lo + _log(rng, 1, 12000 if quant else 4000), "budget": budget, "block": rng.choice([16, 32, 64]),
                "quant": quant}
    return {"op": op, "n": _log(rng, 1, 6000), "q_heads": rng.choice([1, 8, 16, 20, 32]), "k_heads": rng.choice([1, 1, 4, 8]),
            "nope": rng.choice([0, 64, 128]), "rot": rng.choice([32, 64, 64, 96, 128]),
            "layout": rng.choice(["interleaved", "half"]), "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
            "dtype": rng.choice(["f32", "bf16", "f16"]), "transpose": rng.random() < 0.3, "far": _log(rng, 1024, 4000000)}


def lengths(case):
    """The sequences' lengths: log-uniform in [lo, hi], the same for every seed."""
    rng = random.Random("%d %d %d" % (case["n"], case["lo"], case["hi"]))
    return [_log(rng, case["lo"], case["hi"]) for _ in range(case["n"])]


def work(case):
    if case["op"] == "rope":
        size = 4 if case["dtype"] == "f32" else 2
        values = case["n"] * (case["q_heads"] + case["k_heads"]) * case["rot"]
        return {"bytes": 2 * values * size + 4 * case["n"], "flops": 3 * values}
    lens = lengths(case)
    if case["op"] == "mass":
        tokens, queries = sum(lens), case["n"] * case["n_q"] * case["heads"]
        row = W + 2 * BLOCKS if case["quant"] else 4 * W
        return {"bytes": tokens * (row + 8) + queries * (W + 1) * 4 + 4 * sum(-(-x // case["block"]) for x in lens),
                "flops": 2 * tokens * case["n_q"] * case["heads"] * W}
    kept = [min(x, case["budget"]) for x in lens]
    if case["op"] == "select":
        return {"bytes": case["layers"] * 4 * (sum(lens) + sum(kept)), "flops": case["layers"] * sum(lens)}
    row = W + 2 * BLOCKS if case["quant"] else 4 * W
    moved = sum(k for k, x in zip(kept, lens) if k < x)
    return {"bytes": max(4, case["layers"] * (moved * (2 * row + 8) + 4 * sum(kept))), "flops": 0}


# ------------------------------------------------------------------ inputs
class _PoolMemory:
    """Pool memory of the library as a torch tensor sees it; keeps the pool alive."""

    def __init__(self, pool, address, shape, kind):
        self.pool = pool
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (address, False), "version": 3}


def _rows(gen, count, dev):
    return torch.randn(count, W, generator=gen, device=dev)


def _q8(x):
    """Rows of f32 as Q8_0: int8 values and one f16 scale to 32 of them."""
    b = x.view(x.shape[0], BLOCKS, 32)
    d = b.abs().amax(2) / 127.0
    q = torch.where(d[..., None] > 0, (b / d.clamp_min(1e-30)[..., None]).round(), torch.zeros_like(b))
    return q.clamp(-127, 127).to(torch.int8).view(-1, W), d.to(torch.float16)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rope":
        kind = DTYPES[case["dtype"]]
        n, rot = case["n"], case["rot"]
        state["q"] = torch.randn(n, case["q_heads"], case["nope"] + rot, generator=gen, device=dev).to(kind)
        state["k"] = torch.randn(n, case["k_heads"], rot, generator=gen, device=dev).to(kind)
        # consecutive positions of a prompt that ends at the far end
        first = int(torch.randint(0, max(1, case["far"] - n), (1,), generator=gen, device=dev))
        state["positions"] = torch.arange(first, first + n, device=dev, dtype=torch.int32)
        state["q_out"] = torch.empty(n, case["q_heads"], rot, dtype=kind, device=dev)
        state["k_out"] = torch.empty(n, case["k_heads"], rot, dtype=kind, device=dev)
        if own:
            state["rope"] = _kvcu().Rope(rot, layout=case["layout"], base=10000.0, scaling=case["scaling"], factor=16.0,
                                         orig_ctx=4096)
        return state
    lens = lengths(case)
    n = case["n"]
    longest = max(lens)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if case["op"] == "select":
        layers = case["layers"]
        # running sums of attention weights: a few heavy positions, many near nothing, some equal
        mass = torch.randn(layers, n, longest, generator=gen, device=dev).mul_(3.0).exp_()
        mass[torch.rand(mass.shape, generator=gen, device=dev) < 0.1] = 0.0
        state["mass"] = mass
        state["keep"] = torch.empty(layers, n, case["budget"], dtype=torch.int32, device=dev)
        state["counts"] = torch.empty(n, dtype=torch.int32, device=dev)
        if own:
            state["pool"] = _kvcu().DevicePool(0, 1, 1, 16, R, P, True)
        return state
    # the paged cache: blocks in shuffled order, some of them free
    bs, layers = case["block"], case.get("layers", 1)
    per = [-(-x // bs) for x in lens]
    nb = sum(per) + 3
    order = torch.randperm(nb, generator=gen, device=dev)[:sum(per)]
    offsets = [0]
    for x in per:
        offsets.append(offsets[-1] + x)
    state["tables"] = order.to(torch.int32)
    state["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
    total = layers * nb * bs
    if own:
        kvcu = _kvcu()
        pool = state["pool"] = kvcu.DevicePool(0, layers, nb, bs, R, P, case["quant"])
        d = pool.describe()
    if case["quant"]:
        if own:
            state["qs"] = torch.as_tensor(_PoolMemory(pool, d.qs, (total, W), "|i1"), device=dev)
            state["sc"] = torch.as_tensor(_PoolMemory(pool, d.sc, (total, BLOCKS), "<f2"), device=dev)
        else:
            state["qs"] = torch.empty(total, W, dtype=torch.int8, device=dev)
            state["sc"] = torch.empty(total, BLOCKS, dtype=torch.float16, device=dev)
    else:
        if own:
            state["kv"] = torch.as_tensor(_PoolMemory(pool, d.kv, (total, R), "<f4"), device=dev)
            state["pe"] = torch.as_tensor(_PoolMemory(pool, d.pe, (total, P), "<f4"), device=dev)
        else:
            state["kv"] = torch.empty(total, R, device=dev)
            state["pe"] = torch.empty(total, P, device=dev)
    for at in range(0, total, 1 << 18):
        x = _rows(gen, min(1 << 18, total - at), dev)
        if case["quant"]:
            state["qs"][at:at + len(x)], state["sc"][at:at + len(x)] = _q8(x)
        else:
            state["kv"][at:at + len(x)], state["pe"][at:at + len(x)] = x[:, :R], x[:, R:]
    if case["op"] == "compact":
        # kept: any ascending choice of the positions, more of them early and late
        keep = torch.full((layers, n, case["budget"]), -1, dtype=torch.int32, device=dev)
        kept = [min(x, case["budget"]) for x in lens]
        for b in range(n):
            key = torch.rand(layers, lens[b], generator=gen, device=dev)
            key[:, :8] += 1.0
            key[:, -8:] += 1.0
            keep[:, b, :kept[b]] = key.topk(kept[b], dim=1).indices.sort(dim=1).values.to(torch.int32)
        state["keep"] = keep
        state["counts"] = torch.tensor(kept, dtype=torch.int32, device=dev)
        state["mass"] = torch.rand(layers, n, longest, generator=gen, device=dev)
        return state
    state["q"] = torch.randn(n, case["n_q"], case["heads"], W, generator=gen, device=dev)
    state["lse"] = torch.empty(n, case["n_q"], case["heads"], device=dev)
    for b in range(n):
        k, s = _entry_rows(state, b, torch.float32), state["q"][b].view(-1, W)
        s = ((s @ k.T) * SCALE).view(case["n_q"], case["heads"], -1)
        seen = lens[b] - case["n_q"] + 1 + torch.arange(case["n_q"], device=dev)
        s = s.masked_fill(torch.arange(lens[b], device=dev) >= seen[:, None, None], -math.inf)
        state["lse"][b] = torch.logsumexp(s.double(), dim=2)
    # the sum of a few earlier steps
    state["mass"] = torch.rand(n, longest, generator=gen, device=dev) * (4.0 * case["n_q"] * case["heads"] / state["lens"][:, None])
    # the newest rows are not in the running sum yet
    state["old_lens"] = (state["lens"] - case["n_q"]).clamp_min(0)
    if own:
        ws = state["ws"] = kvcu.DecodeWorkspace(0, n, case["heads"])
        ws.plan(pool, state["lens"])
    return state


def _entry_rows(state, b, kind):
    """The cached rows of one sequence in the first layer, as the values they stand for."""
    bs, length = state["case"]["block"], int(state["lens"][b])
    p = torch.arange(length, device=state["lens"].device)
    at = state["tables"][int(state["offsets"][b]) + p // bs].long() * bs + p % bs
    if state["case"]["quant"]:
        q, d = state["qs"][at].to(kind).view(length, BLOCKS, 32), state["sc"][at].to(kind)
        return (q * d[..., None]).view(length, W)
    return torch.cat([state["kv"][at], state["pe"][at]], 1).to(kind)


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"mass": _run_mass, "select": _run_select, "compact": _run_compact, "rope": _run_rope}[case["op"]](state, case)


def _run_mass(state, case):
    if own:
        state["ws"].attn_mass(state["pool"], 0, state["q"], state["lse"], state["offsets"], state["tables"], state["lens"],
                              SCALE, state["mass"], decay=case["decay"], old_lens=state["old_lens"])
        return state["mass"]
    bs, n_q, heads, step = case["block"], case["n_q"], case["heads"], 128
    lens, mass, dev = state["lens"].long(), state["mass"], state["mass"].device
    tiles = (lens + step - 1) // step
    entry = torch.repeat_interleave(torch.arange(len(lens), device=dev), tiles)
    start = (torch.arange(len(entry), device=dev) - (tiles.cumsum(0) - tiles)[entry]) * step
    p = start[:, None] + torch.arange(step, device=dev)
    there = p < lens[entry][:, None]
    q_at = torch.where(there, p, torch.zeros_like(p))
    rows = state["tables"][state["offsets"][entry].long()[:, None] + q_at // bs].long() * bs + q_at % bs
    if case["quant"]:
        k = state["qs"][rows].float().view(-1, step, BLOCKS, 32) * state["sc"][rows].float()[..., None]
        k = k.view(-1, step, W)
    else:
        k = torch.cat([state["kv"][rows], state["pe"][rows]], 2)
    s = torch.bmm(k, state["q"].view(len(lens), n_q * heads, W)[entry].transpose(1, 2)) * SCALE
    w = torch.exp(s - state["lse"].view(len(lens), 1, n_q * heads)[entry]).view(-1, step, n_q, heads).sum(3)
    seen = lens[entry][:, None] - n_q + 1 + torch.arange(n_q, device=dev)
    w = torch.where(p[:, :, None] < seen[:, None, :], w, torch.zeros_like(w)).sum(2)
    old = torch.where(p < state["old_lens"].long()[entry][:, None], case["decay"] * mass[entry[:, None], q_at],
                      torch.zeros_like(w))
    mass[entry[:, None].expand_as(p)[there], p[there]] = (old + w)[there]
    return mass


def _run_select(state, case):
    if own:
        state["pool"].evict_select(state["mass"], state["lens"], case["budget"], case["sink"], case["recent"], state["keep"],
                                   state["counts"])
        return state["keep"], state["counts"]
    mass, lens, budget = state["mass"], state["lens"].long(), case["budget"]
    p = torch.arange(mass.shape[2], device=mass.device)
    key = torch.where((p < case["sink"]) | (p >= lens[:, None] - case["recent"]), torch.full_like(mass, math.inf), mass)
    key = torch.where(p < lens[:, None], key, torch.full_like(mass, -math.inf))
    first = torch.sort(key, dim=2, descending=True, stable=True).indices[:, :, :budget]
    counts = lens.clamp_max(budget)
    nth = torch.arange(first.shape[2], device=mass.device)
    chosen = torch.sort(torch.where(nth < counts[:, None], first, first.new_full((), 1 << 40)), dim=2).values
    keep = torch.full_like(state["keep"], -1)
    keep[:, :, :first.shape[2]] = torch.where(nth < counts[:, None], chosen, chosen.new_full((), -1)).to(torch.int32)
    return keep, counts.to(torch.int32)


def _run_compact(state, case):
    names = ["qs", "sc"] if case["quant"] else ["kv", "pe"]
    if own:
        state["pool"].evict_compact(0, state["offsets"], state["tables"], state["keep"], state["counts"], mass=state["mass"])
        return [state[x] for x in names] + [state["mass"]]
    bs, keep, dev = case["block"], state["keep"].long(), state["mass"].device
    layers, n, budget = keep.shape
    j = torch.arange(budget, device=dev)
    there = (j < state["counts"].long()[:, None]).expand_as(keep)
    layer = torch.arange(layers, device=dev)[:, None, None].expand_as(keep)[there]
    entry = torch.arange(n, device=dev)[:, None].expand_as(keep)[there]
    to, source = j.expand_as(keep)[there], keep[there]
    rows = state[names[0]].shape[0] // layers
    first = state["offsets"][entry].long()

    def at(p):
        return layer * rows + state["tables"][first + p // bs].long() * bs + p % bs

    for x in (state[names[0]], state[names[1]]):
        x[at(to)] = x[at(source)]
    state["mass"][layer, entry, to] = state["mass"][layer, entry, source]
    return [state[x] for x in names] + [state["mass"]]


def _frequencies(case, kind):
    """Angle of a position per step, and the magnitude, of the case's scaling (factor 16, trained to 4096, base 10000)."""
    rot, base, factor, trained = case["rot"], 10000.0, 16.0, 4096
    i = torch.arange(0, rot, 2, dtype=kind, device="cuda")
    if case["scaling"] == "ntk":
        base = base * factor ** (rot / (rot - 2.0))
    f = base ** (-i / rot)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] != "yarn":
        return f, 1.0
    fast, slow = (rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    low, high = max(math.floor(fast), 0), min(math.ceil(slow), rot - 1)
    ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _run_rope(state, case):
    nope = case["nope"]
    if own:
        state["rope"].apply(state["positions"], state["q"][:, :, nope:], state["k"], state["q_out"], state["k_out"],
                            transpose=case["transpose"])
        return state["q_out"], state["k_out"]
    f, magnitude = _frequencies(case, torch.float64)  # far positions' angles need 64 bits
    angle = state["positions"].double()[:, None] * f
    cos, sin = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    if case["transpose"]:
        sin = -sin
    out = []
    for x in (state["q"][:, :, nope:], state["k"]):
        x = x.float()
        if case["layout"] == "half":
            a, b = x[..., :case["rot"] // 2], x[..., case["rot"] // 2:]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        else:
            a, b = x[..., 0::2], x[..., 1::2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        out.append(y.to(DTYPES[case["dtype"]]))
    return out[0], out[1]


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["op"] == "select":
        return None  # whole numbers
    if case["op"] == "rope":
        rot, turns = case["rot"], []
        for i in range(rot // 2):  # radians per position of pair i
            plain = 10000.0 ** (-2.0 * i / rot)
            part = 1.0 if case["scaling"] == "linear" else 0.0  # how much of the pair is stretched 16 times
            if case["scaling"] == "ntk":
                plain *= 16.0 ** (-2.0 * i / (rot - 2))
            if case["scaling"] == "yarn":
                fast = max(0, math.floor(rot / 2 * math.log(4096 / (64 * math.pi), 10000)))
                slow = min(rot - 1, math.ceil(rot / 2 * math.log(4096 / (2 * math.pi), 10000)))
                part = min(1.0, max(0.0, (i - fast) / max(slow - fast, 0.001)))
            turns.append(plain * (1.0 - part * 15.0 / 16.0))
        f = torch.tensor(turns, dtype=torch.float64, device="cuda")
        magnitude = 1.0 + 0.1 * math.log(16.0) if case["scaling"] == "yarn" else 1.0
        turn = magnitude * torch.exp(1j * state["positions"].double()[:, None] * f)
        turn = (turn.conj() if case["transpose"] else turn)[:, None]
        out = []
        for x in (state["q"][:, :, case["nope"]:].double(), state["k"].double()):
            if case["layout"] == "half":
                z = torch.complex(*x.chunk(2, -1)) * turn
                out.append(torch.cat([z.real, z.imag], -1))
            else:
                z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn
                out.append(torch.view_as_real(z).flatten(-2))
        return out[0], out[1]
    lens = lengths(case)
    if case["op"] == "mass":
        if sum(lens) * case["n_q"] * case["heads"] > 1 << 28:
            return None
        mass = state["mass"].double()
        for b in range(case["n"]):
            k, old = _entry_rows(state, b, torch.float64), int(state["old_lens"][b])
            total = torch.zeros(lens[b], dtype=torch.float64, device=k.device)
            for i in range(case["n_q"]):
                seen = lens[b] - (case["n_q"] - 1 - i)
                s = state["q"][b, i].double() @ k[:seen].T * SCALE
                total[:seen] += torch.exp(s - state["lse"][b, i].double()[:, None]).sum(0)
            total[:old] += case["decay"] * mass[b, :old]
            mass[b, :lens[b]] = total
        return mass
    names = ["qs", "sc"] if case["quant"] else ["kv", "pe"]
    bs, keep = case["block"], state["keep"].long()
    nb = state[names[0]].shape[0] // (case["layers"] * bs)
    for b in range(case["n"]):
        kept = min(lens[b], case["budget"])
        table = state["tables"][int(state["offsets"][b]):int(state["offsets"][b + 1])].long()
        row = (table[:, None] * bs + torch.arange(bs, device=table.device)).view(-1)
        for layer in range(case["layers"]):
            for name in names:
                x = state[name][layer * nb * bs:(layer + 1) * nb * bs]
                x[row[:kept]] = x[row[keep[layer, b, :kept]]]
            state["mass"][layer, b, :kept] = state["mass"][layer, b, keep[layer, b, :kept]].clone()
    return [None if state[x].dtype == torch.int8 else state[x].double() for x in names] + [state["mass"].double()]
