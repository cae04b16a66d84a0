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
