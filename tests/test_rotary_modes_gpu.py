"""Rotary positions under torch's other modes: forward-mode differentiation, alone and together with a backward pass."""
import pytest
import torch
from torch.autograd import forward_ad

import kv_plain
from vision_amd.rotary import Rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def rnd(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def bound(x, want, R, a, half):
    """As in test_rotary_gpu.py: 8 u a (|x1| + |x2|) for the arithmetic in 32 bits, half a step for the result's rounding."""
    x = x.double().cpu().abs()
    size = x.clone()
    size[..., :R] = (x[..., :R // 2] + x[..., R // 2:R]).repeat(*[1] * (x.dim() - 1), 2)
    return half * want.abs() + 8 * 2.0 ** -24 * a * size + 1e-37


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_tangents(dtype):
    scaling = {"type": "yarn", "factor": 4.0, "original": 64}
    r = Rotary(48, 40, scaling=scaling, device=DEV)
    f, a = rotary_frequencies(40, scaling=scaling)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    pos = torch.arange(50, 57, device=DEV)
    q, k, tq, tk = rnd((7, 3, 48), 1, dtype), rnd((7, 1, 48), 2, dtype), rnd((7, 3, 48), 3, dtype), rnd((7, 1, 48), 4, dtype)
    want_q, want_k = r(pos, q, k)
    for with_q, with_k in ((True, True), (True, False), (False, True)):
        with forward_ad.dual_level():
            yq, yk = r(pos, forward_ad.make_dual(q, tq) if with_q else q, forward_ad.make_dual(k, tk) if with_k else k)
            for y, plain, has, t in ((yq, want_q, with_q, tq), (yk, want_k, with_k, tk)):
                got = forward_ad.unpack_dual(y)
                assert torch.equal(got.primal, plain) and (got.tangent is not None) == has
                if has:
                    want = kv_plain.rotary(t, pos, f, a, 40, "half")
                    assert ((got.tangent.double().cpu() - want).abs() <= bound(t, want, 40, a, half)).all()
    with forward_ad.dual_level(), torch.no_grad():
        y = forward_ad.unpack_dual(r(pos, forward_ad.make_dual(q, tq)))
        assert torch.equal(y.tangent, r(pos, tq))
    # a tangent that torch keeps without memory
    with forward_ad.dual_level():
        x = forward_ad.make_dual(q, torch._efficientzerotensor(q.shape, dtype=dtype, device=DEV))
        t = forward_ad.unpack_dual(r(pos, x)).tangent
        assert t is None or not t.any()


def test_tangents_against_differences_and_with_a_gradient():
    r = Rotary(32, layout="interleaved", device=DEV)
    pos = torch.arange(9, device=DEV)
    q, d, w = rnd((9, 2, 32), 1).requires_grad_(), rnd((9, 2, 32), 2), rnd((9, 2, 32), 3)
    with forward_ad.dual_level():
        y, t = forward_ad.unpack_dual(r(pos, forward_ad.make_dual(q, d)))
        # linear: a difference over a step of 1 is the derivative; the three turned tensors are off by 8 u (|x1| + |x2|) and half a step
        with torch.no_grad():
            diff = r(pos, q + d) - r(pos, q)
        assert (t - diff).abs().max() <= 64 * 2.0 ** -24 * float(q.detach().abs().max() + d.abs().max())
        g, = torch.autograd.grad((y * w).sum(), q)
    # <w, J d> both ways: 17 u of its size in an element of g and of t
    g64, t64, d64, w64 = (x.detach().double() for x in (g, t, d, w))
    assert abs((g64 * d64).sum() - (t64 * w64).sum()) <= 17 * 2.0 ** -24 * (d64.abs().sum() * w64.abs().max() + w64.abs().sum() * d64.abs().max())
    # a tangent that itself depends on a leaf: the gradient of <w, J d> with respect to d is the turn back of w
    d = d.requires_grad_()
    with forward_ad.dual_level():
        t = forward_ad.unpack_dual(r(pos, forward_ad.make_dual(q.detach(), d))).tangent
        gd, = torch.autograd.grad((t * w).sum(), d)
    assert torch.equal(gd, g)


def test_lazily_negated_queries_and_gradients():
    r, pos = Rotary(16, device=DEV), torch.arange(4, device=DEV)
    z = torch.complex(rnd((4, 2, 16), 1), rnd((4, 2, 16), 2))
    q = z.conj().imag                                        # strides of 2, and the sign apart
    assert q.is_neg() and torch.equal(r(pos, q), r(pos, -z.imag.contiguous()))
    x = rnd((4, 2, 16), 3).requires_grad_()
    g = torch._neg_view(rnd((4, 2, 16), 4))
    got, = torch.autograd.grad(r(pos, x), x, g)
    want, = torch.autograd.grad(r(pos, x), x, g.resolve_neg())
    assert torch.equal(got, want)


@pytest.mark.filterwarnings("ignore")
def test_under_torch_compile():
    """The calls stay calls: what surrounds them may be compiled, the results are the eager ones."""
    from vision_amd.kvcache import KVCache
    r, pos = Rotary(64, device=DEV), torch.arange(6, device=DEV)
    c, table = KVCache(2, 2, 64, device=DEV), torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    start, lengths = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1,), 6, dtype=torch.int32, device=DEV)

    def step(q, k, v):
        q, k = r(pos, q * 2, k)
        c.append(k, v, table, start)
        return c.attend(q, table, lengths) + 1

    q, k, v = rnd((6, 4, 64), 1), rnd((6, 2, 64), 2), rnd((6, 2, 64), 3)
    with torch.no_grad():
        assert torch.equal(torch.compile(step, backend="eager")(q, k, v), step(q, k, v))
    x = q.clone().requires_grad_()
    turn = torch.compile(lambda x: (r(pos, x * 2) ** 2).sum(), backend="eager")
    got, = torch.autograd.grad(turn(x), x)
    want, = torch.autograd.grad((r(pos, x * 2) ** 2).sum(), x)
    assert torch.equal(got, want)
