"""What a column-parallel GatedLinear leaves to the all-reduce of its input gradient, with a test double for the kernels."""
import contextlib

import pytest
import torch

from minitransformer_b200 import kernels
from minitransformer_b200.module import config, gated_linear
from test_norm_gated_cpu import _ExactOp


class _MarginOp(_ExactOp):
    """Records the SMs that each product leaves idle."""

    def __init__(self):
        self.margin, self.seen = 0, []

    @contextlib.contextmanager
    def sm_margin(self, sms):
        before, self.margin = self.margin, sms
        try:
            yield
        finally:
            self.margin = before

    def qgemm(self, *a, **k):
        self.seen.append(self.margin)
        return super().qgemm(*a, **k)


class _Done:
    def wait(self):
        pass


@pytest.mark.parametrize("tp_size,margins", [(1, [0, 0]), (2, [0, 16])])
def test_wgrad_leaves_sms_to_the_all_reduce_of_dgrad(monkeypatch, tp_size, margins):
    monkeypatch.delenv("MT_TP_SM_MARGIN", raising=False)
    monkeypatch.setattr(gated_linear, "allreduce", lambda t, group, async_op: (t, _Done()))
    op = _MarginOp()
    lin = gated_linear.GatedLinear(32, 64, parallel_mode="column", tp_size=tp_size, device="cpu", params_dtype=torch.bfloat16,
                                   qlinear_params=config.QLinearParams(quantize=True, quantize_op=op))
    lin.set_tensor_parallel_group(None)
    x = torch.randn(32, 32).to(torch.bfloat16).requires_grad_()
    lin(x).sum().backward()
    assert op.seen == margins and x.grad is not None and lin.weight.grad is not None


@pytest.mark.parametrize("tp_size,switched", [(1, []), (2, [False])])
def test_tensor_parallel_layers_switch_early_launches_off(monkeypatch, tp_size, switched):
    calls = []
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(kernels, "set_launch_overlap", calls.append)
    gated_linear.GatedLinear(32, 64, parallel_mode="column", tp_size=tp_size, device="meta", params_dtype=torch.bfloat16,
                             qlinear_params=config.QLinearParams(quantize=True, quantize_op=_MarginOp()))
    assert calls == switched
