"""Derivatives that the norm and the gated projection do not have are refused, not lost (test doubles for the kernels)."""
import pytest
import torch
from torch.autograd import forward_ad

from minitransformer_b200 import _lib, kernels
from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear, gated_linear
from minitransformer_b200.module.rmsnorm import RMSNorm
from test_norm_gated_cpu import _ExactOp

BF = torch.bfloat16
EXACT = config.QLinearParams(quantize=True, quantize_op=_ExactOp())
PLAIN = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.NON_QUANTIZE)


@pytest.fixture
def norm(monkeypatch):
    def forward(x, weight, eps=1e-5, *, residual=None, quantize=True, return_transpose=True, want_amax=False):
        h = x if residual is None else x + residual
        rstd = (h.float().square().mean(-1) + eps).rsqrt()
        return kernels.RmsNormResult(h, rstd, (h.float() * rstd[:, None] * weight.float()).to(x.dtype))

    def backward(dy, h, weight, rstd, *, dresidual=None):
        xhat, a = h.float() * rstd[:, None], dy.float() * weight.float()
        dx = rstd[:, None] * (a - xhat * (a * xhat).mean(-1, keepdim=True)) + (0 if dresidual is None else dresidual.float())
        return dx.to(dy.dtype), (dy.float() * xhat).sum(0)

    monkeypatch.setattr(kernels, "rmsnorm", forward)
    monkeypatch.setattr(kernels, "rmsnorm_backward", backward)
    return RMSNorm(32, params_dtype=BF, device="cpu", qlinear_params=PLAIN)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(norm, grad):
    x, r, w = torch.randn(32, 32).to(BF), torch.randn(32, 32).to(BF), torch.randn(64, 32).to(BF)
    lin = GatedLinear(32, 32, device="cpu", params_dtype=BF, qlinear_params=EXACT)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for f in (lambda: norm(dx), lambda: norm(x, dx), lambda: lin(dx), lambda: gated_linear(dx, w, qlinear_params=EXACT),
                  lambda: gated_linear(x, dw, qlinear_params=EXACT)):
            with pytest.raises(_lib.MtError, match="forward-mode"):
                f()
        # without a tangent, and where torch computes, the level changes nothing
        norm(x, r), lin(x)
        assert forward_ad.unpack_dual(gated_linear(dx, w, qlinear_params=PLAIN)).tangent is not None


def test_second_derivatives_are_refused(norm):
    x, r = torch.randn(32, 32).to(BF).requires_grad_(), torch.randn(32, 32).to(BF).requires_grad_()
    lin = GatedLinear(32, 32, device="cpu", params_dtype=BF, qlinear_params=EXACT)
    for f, inputs in ((lambda: norm(x), (x, norm.weight)), (lambda: sum(norm(x, r)), (x, r)), (lambda: lin(x), (x, lin.weight))):
        y = f()
        once = torch.autograd.grad(y.sum(), inputs, retain_graph=True)
        first = torch.autograd.grad(y.sum(), inputs, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(once, first))
        with pytest.raises(_lib.MtError, match="second derivatives"):
            (y.sum() + sum(g.square().sum() for g in first)).backward()
    # gradients that are not differentiated again may have been taken with create_graph
    lin(x).sum().backward(create_graph=True)
    assert x.grad is not None and lin.weight.grad is not None
    # the residual stream alone is an addition, with all its derivatives
    x.grad = None
    first, = torch.autograd.grad(norm(x, r)[1].square().sum(), x, create_graph=True)
    first.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2))
