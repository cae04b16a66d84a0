"""Rotary positions (csrc/rotary.hip) against their formula in 64 bits.

Tolerance: y = a (x1 c - x2 s) in fp32: c and s are off by 3 u (u = 2^-24: the reduced angle's two roundings, the polynomial) and
one more for the amplitude, two products and a sum by one each: 8 u a (|x1| + |x2|); the result's own rounding is half a step."""
import pytest
import torch

import kv_plain
from vision_amd.rotary import Rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def rnd(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def close(y, x, positions, r, scaling=None, inverse=False):
    f, a = rotary_frequencies(r.rotary_dim, scaling=scaling)
    want = kv_plain.rotary(x, positions, f, a, r.rotary_dim, r.layout, inverse)
    y, x = y.detach().double().cpu(), x.detach().double().cpu()
    R = r.rotary_dim
    assert torch.equal(y[..., R:], x[..., R:])
    if r.layout == "half":
        size = (x[..., :R // 2].abs() + x[..., R // 2:R].abs()).repeat(*[1] * (x.dim() - 1), 2)
    else:
        size = (x[..., 0:R:2].abs() + x[..., 1:R:2].abs()).repeat_interleave(2, -1)
    bound = HALF[y_type[0]] * want[..., :R].abs() + 8 * 2.0 ** -24 * a * size + 1e-37
    worst = ((y[..., :R] - want[..., :R]).abs() / bound).max()
    assert worst <= 1, worst


y_type = [None]


@pytest.fixture(params=[torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def dtype(request):
    y_type[0] = request.param
    return request.param


SHAPES = [  # tokens, q heads, k heads, head dim, turned
    (1, 8, 8, 64, 64), (1, 1, 1, 2, 2), (49, 4, 1, 64, 32), (7, 3, 3, 48, 20), (5, 5, 1, 80, 6), (33, 2, 2, 96, 64), (3, 9, 3, 256, 256),
    (1000, 12, 4, 128, 128), (13, 3, 1, 9, 8), (17, 1, 1, 112, 14),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_forward_and_gradient(shape, layout, dtype):
    n, hq, hk, D, R = shape
    r = Rotary(D, R, layout=layout, device=DEV)
    pos = torch.arange(n, device=DEV) + 100
    q, k = rnd((n, hq, D), dtype, 1).requires_grad_(), rnd((n, hk, D), dtype, 2).requires_grad_()
    yq, yk = r(pos, q, k)
    close(yq, q, pos, r)
    close(yk, k, pos, r)
    gq, gk = rnd((n, hq, D), dtype, 3), rnd((n, hk, D), dtype, 4)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    close(dq, gq, pos, r, inverse=True)
    close(dk, gk, pos, r, inverse=True)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 4.0, "original": 4096}], ids=lambda s: s["type"])
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_scaled_and_far_positions(scaling, ptype, dtype):
    r = Rotary(64, scaling=scaling, device=DEV)
    pos = torch.tensor([0, 1, -1, 4095, 4096, 131071, 1000003, 2 ** 31 - 1, -2 ** 31], dtype=ptype, device=DEV)
    q = rnd((9, 2, 64), dtype)
    # at 2^31 the oracle's own float64 product rounds the angle by 2^31 * 2^-53 = 2^-22 radians: compare up to 2^21 exactly
    y = r(pos, q)
    keep = pos.abs() < 2 ** 21
    close(y[keep], q[keep], pos[keep], r, scaling)
    norm = (y.double() ** 2).sum(-1).sqrt() / (q.double() ** 2).sum(-1).sqrt() / r.amplitude
    assert (norm - 1).abs().max() < 2 ** -7
    # far positions: an angle is additive, turning by p and then by -p is the identity
    if r.amplitude == 1.0:
        back = r(-pos[:-1], y[:-1])
        assert (back - q[:-1]).abs().max() <= 4 * HALF[dtype] * q.abs().max() + 1e-5


def test_layouts_in_memory(dtype):
    """Heads before tokens, slices of a fused projection, batches whose leading dimensions do not merge, a lone leading dimension,
    positions that broadcast, expanded and unaligned tensors."""
    D = 32
    r = Rotary(D, 24, device=DEV)
    pos = torch.arange(6, device=DEV)
    heads_first = rnd((2, 3, 6, D), dtype).transpose(1, 2)                                   # [B, T, H, D] over [B, H, T, D]
    y = r(pos, heads_first)
    assert y.stride() == heads_first.stride()
    close(y, heads_first, pos, r)
    qkv = rnd((2, 6, 5 * D + 3), dtype)[..., 3:].unflatten(-1, (5, D))                       # rows not 16-byte aligned
    yq, yk = r(pos, qkv[..., :3, :], qkv[..., 3:4, :])
    close(yq, qkv[..., :3, :], pos, r)
    close(yk, qkv[..., 3:4, :], pos, r)
    one = rnd((1, 1, 1, D), dtype).expand(2, 6, 3, D)
    close(r(pos, one), one, pos, r)
    single = rnd((4, D), dtype)
    close(r(torch.tensor(5, device=DEV), single), single, torch.tensor(5), r)
    many = rnd((2, 3, 2, 6, 2, D), dtype).transpose(0, 2)                                    # leading dims that merge nowhere
    close(r(pos, many), many, pos, r)
    strided = rnd((6, 2, 2 * D), dtype)[..., ::2]                                            # features not adjacent: copied
    close(r(pos, strided), strided, pos, r)
    mixed = rnd((2, 3, 4, 2, D), dtype)
    other = rnd((4, 3, 2, 2, D), dtype).transpose(0, 2)
    p5 = torch.arange(24, device=DEV).view(2, 3, 4)
    yq, yk = r(p5, mixed, other)                                                             # the two merge differently
    close(yq, mixed, p5, r)
    close(yk, other, p5, r)


def test_in_place(dtype):
    r = Rotary(64, 48, layout="interleaved", device=DEV)
    pos = torch.arange(10, device=DEV, dtype=torch.int32)
    qkv = rnd((10, 8, 64), dtype)
    kept = qkv.clone()
    q, k = qkv[:, :4], qkv[:, 4:6]
    wq, wk = r(pos, q, k)
    oq, ok = r.apply_(pos, q, k)
    assert oq is q and ok is k and torch.equal(q, wq) and torch.equal(k, wk) and torch.equal(qkv[:, 6:], kept[:, 6:])
    with pytest.raises(ValueError, match="in place"):
        r.apply_(pos, rnd((1, 1, 64), dtype).expand(10, 2, 64))
    with pytest.raises(ValueError, match="same memory"):
        r.apply_(pos, q, q)
    with pytest.raises(ValueError, match="same memory"):
        r.apply_(pos, q, qkv[:, 3:5])
    with pytest.raises(RuntimeError, match="gradient"):
        r.apply_(pos, kept.requires_grad_())
    # autograd notices what was overwritten
    x = rnd((10, 2, 64), dtype).requires_grad_()
    h = x * 2
    z = (h * h).sum()
    with torch.no_grad():
        r.apply_(pos, h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_empty(dtype):
    r = Rotary(32, device=DEV)
    pos = torch.zeros(0, dtype=torch.int64, device=DEV)
    yq, yk = r(pos, rnd((0, 2, 32), dtype), rnd((0, 1, 32), dtype))
    assert yq.shape == (0, 2, 32) and yk.shape == (0, 1, 32)
    p3 = torch.arange(3, device=DEV)
    q, none = rnd((3, 2, 32), dtype), rnd((3, 0, 32), dtype)
    yq, yk = r(p3, q, none)
    close(yq, q, p3, r)
    assert yk.shape == (3, 0, 32)
    kept = q.clone()
    r.apply_(p3, q, none)
    assert torch.equal(q, yq) and not torch.equal(q, kept)


def test_gradient_against_differences_and_twice():
    y_type[0] = torch.float32
    r = Rotary(16, 12, scaling={"type": "yarn", "factor": 2.0, "original": 64}, device=DEV)
    pos = torch.tensor([3, 70, 9], device=DEV)
    q, k, g = rnd((3, 2, 16), torch.float32).requires_grad_(), rnd((3, 1, 16), torch.float32, 1).requires_grad_(), rnd((3, 2, 16), torch.float32, 2)
    yq, yk = r(pos, q, k)
    loss = (yq * g).sum() + (yk ** 2).sum()
    dq, dk = torch.autograd.grad(loss, (q, k), create_graph=True)
    d = rnd((3, 2, 16), torch.float32, 5)
    with torch.no_grad():                                    # the map is linear: a difference over any step is its derivative
        diff = ((r(pos, q + d) - r(pos, q)) * g).sum()
    assert abs(float((dq * d).sum() - diff)) < 1e-4
    # d/dk |turn k|^2 = 2 a^2 k on the turned part, 2 k behind it
    want = 2 * k.detach() * torch.cat([torch.full((12,), r.amplitude ** 2), torch.ones(4)]).to(DEV)
    assert (dk - want).abs().max() < 1e-5
    again, = torch.autograd.grad((dk ** 2).sum(), k)
    assert (again - 2 * want * want / k.detach()).abs().max() < 1e-3
    # one of the two unused, one not asked for
    yq, yk = r(pos, q, k)
    only, none = torch.autograd.grad(yq.sum(), (q, k), allow_unused=True)
    assert only is not None and none is None
    yq, yk = r(pos, q.detach(), k)
    (yk.sum() + yq.sum()).backward()
    close(k.grad, torch.ones_like(k), pos, r, {"type": "yarn", "factor": 2.0, "original": 64}, inverse=True)


def test_streams_and_graphs(dtype):
    r = Rotary(64, device=DEV)
    pos, q, k = torch.arange(200, device=DEV), rnd((200, 4, 64), dtype), rnd((200, 2, 64), dtype, 1)
    want = r(pos, q, k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = r(pos, q, k)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = r(pos, q, k)
    for shift in (0, 5, 11):
        pos.copy_(torch.arange(200, device=DEV) + shift)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r(pos, q, k), got))


def test_captured_backward(dtype):
    r = Rotary(32, device=DEV)
    pos = torch.arange(20, device=DEV)
    q, g = rnd((20, 2, 32), dtype).requires_grad_(), rnd((20, 2, 32), dtype, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(r(pos, q), q, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, = torch.autograd.grad(r(pos, q), q, g)
    for seed in range(3):
        g.copy_(rnd((20, 2, 32), dtype, seed + 10))
        graph.replay()
        torch.cuda.synchronize()
        close(dq, g, pos, r, inverse=True)


def test_many_tokens():
    """More than 2^31 elements: offsets pass 32 bits."""
    y_type[0] = torch.bfloat16
    r = Rotary(256, device=DEV)
    n = 2 ** 31 // 2048 + 3
    q = torch.empty((n, 8, 256), dtype=torch.bfloat16, device=DEV).normal_()
    pos = torch.arange(n, device=DEV)
    y = r(pos, q)
    for i in (0, 1, n // 2, n - 2, n - 1):
        close(y[i:i + 1], q[i:i + 1], pos[i:i + 1], r)
