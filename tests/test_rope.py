"""kvcu_rope's frequencies and refusals (host only, no GPU): the plain, linear,
NTK and YaRN formulas against numpy, and every description it must turn down."""
import math

import numpy as np
import pytest

import kvcu


def _want(rot, base, scaling, factor, orig, fast=32.0, slow=1.0):
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2.0))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    pair = [rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
    low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
    ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


@pytest.mark.parametrize("rot", [2, 32, 64, 96, 256])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("base,factor,orig", [(10000.0, 16.0, 4096), (500000.0, 8.0, 8191), (10000.0, 1.0, 1)])
def test_frequencies(rot, scaling, base, factor, orig):
    if scaling == "ntk" and rot == 2:
        with pytest.raises(kvcu.KVCudaError):
            kvcu.Rope(rot, scaling=scaling, base=base, factor=factor, orig_ctx=orig)
        return
    r = kvcu.Rope(rot, scaling=scaling, base=base, factor=factor, orig_ctx=orig)
    f, m = r.frequencies()
    wf, wm = _want(rot, base, scaling, factor, orig)
    # a few 64-bit roundings of pow and log (ulp 2.2e-16 each, amplified by the exponent's size, < 20)
    assert np.allclose(f, wf, rtol=1e-13, atol=0)
    assert m == pytest.approx(wm, rel=1e-14)


def test_given_magnitude_and_betas():
    r = kvcu.Rope(64, scaling="yarn", factor=4.0, orig_ctx=4096, beta_fast=16.0, beta_slow=2.0, mscale=0.75)
    f, m = r.frequencies()
    assert m == 0.75
    assert np.allclose(f, _want(64, 10000.0, "yarn", 4.0, 4096, 16.0, 2.0)[0], rtol=1e-13)


@pytest.mark.parametrize("kw", [
    {"rot_dim": 0}, {"rot_dim": 3}, {"rot_dim": 258}, {"base": 1.0}, {"base": float("nan")}, {"base": float("inf")},
    {"scaling": "linear", "factor": 0.5}, {"scaling": "ntk", "factor": float("nan")},
    {"scaling": "yarn", "factor": 4.0, "orig_ctx": 0},
    {"scaling": "yarn", "factor": 4.0, "orig_ctx": 4096, "beta_fast": 1.0, "beta_slow": 2.0},
    {"scaling": "yarn", "factor": 4.0, "orig_ctx": 4096, "beta_slow": -1.0},
    {"mscale": float("nan")}, {"mscale": -1.0},
])
def test_refused_descriptions(kw):
    with pytest.raises(kvcu.KVCudaError) as e:
        kvcu.Rope(**{"rot_dim": 64, **kw})
    assert e.value.name == "InvalidArgument"


def test_refused_names():
    with pytest.raises(ValueError):
        kvcu.Rope(64, layout="other")
    with pytest.raises(ValueError):
        kvcu.Rope(64, scaling="other")


def test_null_handles():
    L = kvcu.lib()
    assert L.kvcu_rope_create(None) is None
    assert L.kvcu_rope_destroy(None) == 0
    assert L.kvcu_rope_frequencies(None, None, None) == -11
    none = (None, 0, 0, 0, None, 0, 0)
    assert L.kvcu_rope_apply(None, 0, 0, 0, 1, None, *none, *none, None) == -11
    r = kvcu.Rope(64)
    assert L.kvcu_rope_apply(r.handle, 0, 3, 0, 1, None, *none, *none, None) == -11  # dtype
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 1, None, *none, *none, None) == 0    # no heads
    q = (0x1000, 4, 256, 64, 0x2000, 256, 64)
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 0, None, *q, *none, None) == 0       # no tokens
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 2, None, *q, *none, None) == -11     # no positions
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 2, 0x100, None, 4, 256, 64, 0x2000, 256, 64, *none, None) == -11
    # overlapping outputs: heads closer than a segment, tokens inside one another's heads, a repeated output
    for out in ((256, 32), (128, 64), (0, 64), (256, 0)):
        assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 2, 0x100, *q[:4], 0x2000, *out, *none, None) == -11, out
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 2, 0x100, 0x1002, *q[1:], *none, None) == -11  # alignment
    assert L.kvcu_rope_apply(r.handle, 0, 0, 0, 2, 0x100, 0x1000, 16385, 64 * 16385, 64, 0x2000, 64 * 16385, 64, *none,
                             None) == -16
