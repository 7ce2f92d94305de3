"""`RMSNorm` with the residual addition in front of it, ready for the quantized linear that follows.

y = h / sqrt(mean(h^2) + eps) * weight with h = x + residual. With `emit_quantized` the same kernel
also quantizes y for the next layer: `output_meta` then goes into that layer's `inp_meta` and its
quantize pass falls away (MXFP8: the copies themselves; NVFP4: max |y|, which saves the abs-max
pass where the Hadamard transform does not need one of its own). Takes the place of the norm in the
reference's unfused LayerNormLinear (miniTransformer/module/layernorm_linear.py:299-306)."""
from typing import Optional

import torch

from . import config
from ._common import first_derivatives_only, refuse_tangents
from .. import kernels
from ..ops import quantization
from ..ops.mxfp8_quantize_op import Mxfp8QuantizeOp, as_quantize_result


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, copies, is_grad_enabled, meta):
        """copies: None, "mxfp8" or "amax"; meta (a QuantizeInputMeta or None) receives them."""
        shape = x.shape
        x2 = x.reshape(-1, shape[-1])
        r2 = None if residual is None else residual.reshape(-1, shape[-1])
        # transposed copies feed a wgrad GEMM, which contracts over the tokens in steps of 16
        transpose = is_grad_enabled and x2.shape[0] % 16 == 0
        r = kernels.rmsnorm(x2, weight, eps, residual=r2, quantize=copies == "mxfp8", return_transpose=transpose,
                            want_amax=copies == "amax")
        if meta is not None:
            meta.amax = r.amax
            if r.quantized is not None:
                meta.quantized = as_quantize_result(r.quantized)
        if is_grad_enabled:
            ctx.shape, ctx.has_residual = shape, residual is not None
            ctx.set_materialize_grads(False)      # a residual stream that leads nowhere costs no zeros
            ctx.save_for_backward(r.h, weight, r.rstd)
        y = r.y.view(shape)
        return y if residual is None else (y, r.h.view(shape))

    @staticmethod
    @first_derivatives_only("RMSNorm")
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        cols = ctx.shape[-1]
        if dy is None:                            # only the residual stream was used
            return (dh, dh if ctx.has_residual else None) + (None,) * 5
        dres = None if dh is None else dh.reshape(-1, cols)
        dx, dweight = kernels.rmsnorm_backward(dy.reshape(-1, cols), h, weight, rstd, dresidual=dres)
        dx = dx.view(ctx.shape)
        return (dx, dx if ctx.has_residual else None, dweight.to(weight.dtype)) + (None,) * 4


class RMSNorm(torch.nn.Module):
    """`weight` [hidden_size]. forward(x) -> y; forward(x, residual) -> (y, h), h = x + residual being the
    residual stream from here on. bf16 activations, hidden_size a multiple of 8 (of 32 with MXFP8
    copies) up to 32768, weight in bf16 or fp32.

    emit_quantized (attribute, off by default): `output_meta` holds what the recipe's quantizer can take
    over for y, for the next layer's `inp_meta`; MXFP8 copies live as long as the y they belong to. qlinear_params: that layer's recipe; if None it is
    taken from QAT_PARAMS the first time it is needed."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, params_dtype: Optional[torch.dtype] = None, device="cuda",
                 qlinear_params: Optional[config.QLinearParams] = None) -> None:
        super().__init__()
        dtype = torch.get_default_dtype() if params_dtype is None else params_dtype
        self.hidden_size, self.eps = hidden_size, eps
        self.weight = torch.nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))
        self.qlinear_params = qlinear_params
        self.emit_quantized = False
        self.output_meta: Optional[quantization.QuantizeInputMeta] = None

    def _copies(self) -> Optional[str]:
        if not self.emit_quantized:
            return None
        if self.qlinear_params is None:
            self.qlinear_params = config.get_qlinear_params_from_env_qat_params()
        if not self.qlinear_params.quantize:
            return None
        return "mxfp8" if isinstance(self.qlinear_params.quantize_op, Mxfp8QuantizeOp) else "amax"

    @torch._dynamo.disable(recursive=True)
    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if residual is not None and residual.shape != x.shape:
            raise kernels._lib.MtError(f"residual of shape {tuple(residual.shape)} for x of shape {tuple(x.shape)}")
        refuse_tangents("RMSNorm", x, residual, self.weight)
        copies = self._copies()
        self.output_meta = quantization.QuantizeInputMeta() if copies else None
        grad = torch.is_grad_enabled() and (x.requires_grad or self.weight.requires_grad or
                                            (residual is not None and residual.requires_grad))
        meta = self.output_meta
        args = (x, residual, self.weight, self.eps, copies, grad, meta)
        out = _RMSNorm.apply(*args) if grad else _RMSNorm.forward(None, *args)
        if meta is not None and meta.quantized is not None:
            meta.quantized = quantization.TensorCopies(out if residual is None else out[0], meta.quantized)
        return out
