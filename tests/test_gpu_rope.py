"""kvcu_rope_apply on the GPU against the rotation in 64 bits.

Tolerances: the reduced angle is rounded to f32 once (2^-24 of half a turn's pi),
the sine and cosine, their product with the magnitude, the two products and the
sum each by half a unit: together under 8 * 2^-24 of m (|x_a| + |x_b|) in f32; an
output of 16 bits is rounded once more (half a step of its type, and the same f32 error)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    import torch

    import kvcu

    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    kvcu.init(0)
    return kvcu


def _want(x, pos, f, m, layout, transpose):
    import torch

    f = torch.from_numpy(f).to(x.device)
    turn = m * torch.exp(1j * pos.double()[:, None, None] * f)
    turn = turn.conj() if transpose else turn
    x = x.double()
    if layout == "half":
        z = torch.complex(*x.chunk(2, -1)) * turn
        y, a = torch.cat([z.real, z.imag], -1), x.abs()
        a = (a.chunk(2, -1)[0] + a.chunk(2, -1)[1]).repeat(1, 1, 2)
    else:
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn
        y = torch.view_as_real(z).flatten(-2)
        a = x.abs().reshape(*x.shape[:-1], -1, 2).sum(-1).repeat_interleave(2, -1)
    return y, m * a


def _check(got, x, pos, f, m, layout, transpose=False):
    import torch

    want, mag = _want(x, pos, f, m, layout, transpose)
    # f / 2 pi, its product with pos and the reference's own pos * f are 64-bit roundings: 2^-53 of the angle each
    tol = (8 * 2.0 ** -24 + pos.double()[:, None, None] * 2.0 ** -51) * mag
    if got.dtype != torch.float32:
        # half a step of the type relative to the value, and its smallest step (f16 subnormals)
        tol = tol + (torch.finfo(got.dtype).eps / 2 * want.abs()).clamp_min(2.0 ** -25 if got.dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("rot,nope,qh,kh,n", [(64, 128, 20, 1, 1), (64, 0, 20, 1, 333), (2, 1, 3, 1, 7), (96, 64, 8, 8, 65),
                                              (128, 0, 1, 4, 1000), (256, 8, 5, 2, 17), (10, 3, 2, 1, 50)])
def test_against_64_bits(kv, dtype, layout, rot, nope, qh, kh, n):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rot * 1000 + n)
    dt = getattr(torch, dtype)
    q = torch.randn(n, qh, nope + rot, device="cuda", generator=g).to(dt)
    k = torch.randn(n, kh, rot, device="cuda", generator=g).to(dt)
    pos = torch.randint(0, 2 ** 31 - 1, (n,), device="cuda", generator=g).to(torch.int32)
    pos[0] = 0
    kinds = ["none", "linear", "yarn"] + (["ntk"] if rot > 2 else [])
    for scaling in kinds:
        for transpose in (False, True):
            r = kv.Rope(rot, layout=layout, scaling=scaling, factor=16.0, orig_ctx=4096)
            f, m = r.frequencies()
            qo = torch.full((n, qh, rot), float("nan"), device="cuda", dtype=dt)
            ko = torch.full((n, kh, rot), float("nan"), device="cuda", dtype=dt)
            r.apply(pos, q[:, :, nope:], k, qo, ko, transpose=transpose)
            _check(qo, q[:, :, nope:], pos, f, m, layout, transpose)
            _check(ko, k, pos, f, m, layout, transpose)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_in_place_part_of_the_head_only(kv, layout):
    import torch

    q = torch.randn(50, 20, 192, device="cuda")
    before = q.clone()
    pos = torch.arange(1000, 1050, device="cuda", dtype=torch.int32)
    r = kv.Rope(64, layout=layout)
    f, m = r.frequencies()
    r.apply(pos, q[:, :, 128:])
    assert torch.equal(q[:, :, :128], before[:, :, :128])
    _check(q[:, :, 128:], before[:, :, 128:], pos, f, m, layout)
    # a rotation of magnitude 1 and its transpose give the input back (two roundings each way)
    r.apply(pos, q[:, :, 128:], transpose=True)
    assert (q - before).abs().max() <= 32 * 2.0 ** -24 * before.abs().max()


def test_strides_orders_and_rows_around(kv):
    """Heads outside tokens, an input that repeats one head, an unaligned output (the scalar
    path) and rows behind the batch, which stay as they were."""
    import torch

    n, h, rot = 37, 6, 64
    pos = torch.randint(0, 100000, (n,), device="cuda").to(torch.int32)
    r = kv.Rope(rot, layout="half", scaling="yarn", factor=4.0, orig_ctx=4096)
    f, m = r.frequencies()
    x = torch.randn(h, n, rot, device="cuda").transpose(0, 1)
    y = torch.zeros(h, n + 3, rot, device="cuda")
    r.apply(pos, x, q_out=y.transpose(0, 1)[:n])
    _check(y.transpose(0, 1)[:n], x, pos, f, m, "half")
    assert (y[:, n:] == 0).all()
    one = torch.randn(n, 1, rot, device="cuda").expand(n, h, rot)
    buf = torch.zeros(n * h * (rot + 1) + 1, device="cuda")
    out = buf[1:].view(n, h, rot + 1)[:, :, :rot]
    r.apply(pos, one, q_out=out)
    _check(out, one, pos, f, m, "half")
    assert buf[0] == 0 and (buf[1:].view(n, h, rot + 1)[:, :, rot] == 0).all()


def test_gradient_by_autograd_and_by_differences(kv):
    """The transposed call is the gradient of the forward call: against autograd through the
    plain rotation in 64 bits, and against central differences of the forward call itself."""
    import torch

    n, h, rot = 9, 3, 32
    r = kv.Rope(rot, scaling="yarn", factor=8.0, orig_ctx=2048)
    f, m = r.frequencies()
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(n, h, rot, device="cuda", generator=g)
    dy = torch.randn(n, h, rot, device="cuda", generator=g)
    pos = torch.randint(0, 50000, (n,), device="cuda", generator=g).to(torch.int32)
    dx = torch.empty_like(x)
    r.apply(pos, dy, q_out=dx, transpose=True)
    x64 = x.double().requires_grad_()
    fd = torch.from_numpy(f).cuda()
    ang = pos.double()[:, None, None] * fd
    a, b = x64[..., 0::2], x64[..., 1::2]
    y = torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2) * m
    (y * dy.double()).sum().backward()
    assert (dx.double() - x64.grad).abs().max() <= 16 * 2.0 ** -24 * m * dy.abs().max()
    # differences: the map is linear, so a step of 1 has no truncation error, only roundings
    for (t, hh, e) in ((0, 0, 0), (3, 1, 7), (8, 2, 31)):
        ys = []
        for s in (0.5, -0.5):
            xs = x.clone()
            xs[t, hh, e] += s
            out = torch.empty_like(x)
            r.apply(pos, xs, q_out=out)
            ys.append((out.double() * dy.double()).sum())
        assert abs(float(ys[0] - ys[1]) - float(dx[t, hh, e])) <= 64 * 2.0 ** -24 * m * float(x.abs().max() * dy.abs().max())


def test_plain_form_is_the_references(kv):
    """The reference's own rotation (src/math.zig:197-240, pairs (2i, 2i+1)) at small positions."""
    import torch

    import mla_ref

    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 2, 64)).astype(np.float32)
    pos = np.array([0, 1, 5, 63, 200], np.int32)
    r = kv.Rope(64)
    t = torch.from_numpy(x).cuda()
    r.apply(torch.from_numpy(pos).cuda(), t)
    got = t.cpu().numpy()
    for i in range(5):
        for h in range(2):
            # the reference rounds the angle itself to f32: up to 200 * 2^-23 rad at these positions
            assert np.allclose(got[i, h], mla_ref.rope_apply(x[i, h], int(pos[i]), 64, 10000.0), atol=200 * 2.0 ** -23 * 8)


def test_side_stream_and_graph(kv):
    import torch

    n, h, rot = 64, 20, 64
    r = kv.Rope(rot)
    f, m = r.frequencies()
    x, y = torch.randn(n, h, rot, device="cuda"), torch.empty(n, h, rot, device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r.apply(pos, x, q_out=y, stream=s)
    s.synchronize()
    _check(y, x, pos, f, m, "interleaved")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.apply(pos, x, q_out=y, stream=torch.cuda.current_stream())
    x.normal_()
    pos += 777
    graph.replay()
    torch.cuda.synchronize()
    _check(y, x, pos, f, m, "interleaved")


def test_refused_tensors(kv):
    import torch

    r = kv.Rope(64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        r.apply(pos, x[:, :, :32])
    with pytest.raises(ValueError):
        r.apply(pos.long(), x)
    with pytest.raises(ValueError):
        r.apply(pos, x.double())
    with pytest.raises(ValueError):
        r.apply(pos, x, q_out=torch.zeros(4, 2, 64))
    with pytest.raises(ValueError):
        r.apply(pos, x, k=x.half())
    with pytest.raises(kv.KVCudaError):
        r.apply(pos, x, q_out=x[:1].expand(4, 2, 64))
    r.apply(pos)  # nothing to rotate
    r.apply(pos[:0], x[:0])


def test_positions_are_whole_numbers_and_may_be_one_of_many(kv):
    import torch

    rope = kv.Rope(64)
    x = torch.randn(1, 3, 64, device="cuda")
    with pytest.raises(ValueError):
        rope.apply(torch.ones(1, device="cuda"), q=x)
    with pytest.raises(ValueError):
        rope.apply(torch.ones(1, dtype=torch.int64, device="cuda"), q=x)
    many = torch.tensor([7, 8, 9, 10], dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(x), torch.empty_like(x)
    rope.apply(many[1:2], q=x, q_out=a)
    rope.apply(many[::4] + 1, q=x, q_out=b)  # a stride of its own, but one position
    torch.cuda.synchronize()
    assert torch.equal(a, b)
