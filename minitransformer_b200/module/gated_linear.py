"""`GatedLinear`: the first half of a gated feed-forward block, h = act(x Wg^T) * (x Wu^T), as one layer.

Both projections, the activation and the product run in one block-scaled GEMM kernel; the backward
pass computes the gradients of activation and product and quantizes them in one pass, then uses the
GEMMs of `Linear`:
  forward   [g | u] = q(x) . q(W)^T,  h = act(g) * u           W = [Wg; Wu], one weight of 2F rows
  dgrad     dx = q([dg | du]) . q(W^T copy)^T                  contraction over 2F
  wgrad     dW = q([dg | du]^T copy) . q(x^T copy)^T           contraction over tokens
Quantization, the weight cache across microbatches and the `main_grad` protocol are those of `Linear`
(miniTransformer/module/linear.py:198-460); tensor parallelism is that of `GroupedLinear`: column
parallel, an all-reduce of dgrad, no sequence parallelism."""
import logging
from typing import Callable, Optional, Union

import torch

from . import config
from ._common import first_derivatives_only, refuse_tangents
from .base import LayerLinearBaseModule
from .linear import _overlap_sm_margin, _QuantizedLinear, _sm_margin
from .. import kernels
from ..distributed.distributed import allreduce, set_tensor_model_parallel_attributes
from ..ops import quantization
from ..ops.mxfp8_quantize_op import as_quantize_result
from ..utils.utils import cast_if_needed, divide, is_rank_0

logger = logging.getLogger(__name__)

_NUM_FN_ARGS = 14


def _pad_rows(t: torch.Tensor, rows: int) -> torch.Tensor:
    return t if t.shape[0] == rows else torch.nn.functional.pad(t, (0, 0, 0, rows - t.shape[0]))


class _QuantizedGatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, x_meta, w, weight_qresult_cache, activation, tp_group, tp_size, parallel_mode, qlinear_params,
                activation_dtype, is_grad_enabled, is_first_microbatch, fuse_wgrad_accumulation, out_meta):
        """weight_qresult_cache: None (nothing kept) or a QuantizeResultCache. out_meta: None, or (a QuantizeInputMeta that receives what the next layer's quantizer can take over,
        whether that is the MXFP8 copy of h)."""
        op = qlinear_params.quantize_op
        assert op is not None and hasattr(op, "gated_qgemm"), "the recipe's backend has no gated projection"
        if activation_dtype != torch.bfloat16:
            raise kernels._lib.MtError(f"GatedLinear computes in bf16, got {activation_dtype} activations")
        x_shape = x.shape
        x = cast_if_needed(x.reshape(-1, x_shape[-1]), activation_dtype)
        M = x.shape[0]
        # The wgrad GEMM contracts over the tokens in whole 32-blocks: a ragged batch is continued with rows of
        # zeros, which add nothing to any gradient (and an empty one becomes 32 of them).
        rows = max(1, (M + 31) // 32) * 32 if is_grad_enabled else M
        if rows != M:
            x, x_meta = _pad_rows(x, rows), None
        qres_x = op.quantize(x, qlinear_params.x_params, return_transpose=is_grad_enabled, input_meta=x_meta)

        # (a cache filled under no_grad holds no transposed copy: refill it before a training pass)
        cache = weight_qresult_cache
        usable = cache is not None and cache.data is not None and not (is_grad_enabled and cache.data_t is None)
        keep = usable and bool(getattr(cache, "keep", False))
        if not keep and (is_first_microbatch or is_first_microbatch is None or not usable):
            qres_w = op.quantize(w, qlinear_params.w_params, return_transpose=is_grad_enabled)
            if cache is not None:
                cache.store(qres_w)
        else:
            qres_w = cache.to_qresult()

        meta, copy = out_meta if out_meta is not None else (None, False)
        r = op.gated_qgemm(qres_x.data, qres_w.data, qres_x.scale, qres_w.scale, activation,
                           global_amax_qx=qres_x.global_amax_row, global_amax_qw=qres_w.global_amax_row,
                           want_gu=is_grad_enabled, quantize_h=copy and rows == M, want_amax=meta is not None and not copy)
        if meta is not None:
            meta.amax = r.amax
            if r.quantized is not None:
                meta.quantized = as_quantize_result(r.quantized)
        if is_grad_enabled:
            ctx.tp_group, ctx.tp_size, ctx.parallel_mode, ctx.x_shape = tp_group, tp_size, parallel_mode, x_shape
            ctx.rows, ctx.activation, ctx.qlinear_params, ctx.quantize_op = rows, activation, qlinear_params, op
            ctx.is_first_microbatch, ctx.fuse_wgrad_accumulation = is_first_microbatch, fuse_wgrad_accumulation
            ctx.sx_t_swz, ctx.sw_t_swz = qres_x.scale_t_swz, qres_w.scale_t_swz
            ctx.save_for_backward(qres_x.data_t, qres_x.scale_t, qres_x.global_amax_col, qres_w.data_t, qres_w.scale_t,
                                  qres_w.global_amax_col, r.gu, w)
        return r.h[:M].view(*x_shape[:-1], r.h.shape[-1])

    @staticmethod
    @first_derivatives_only("GatedLinear")
    def backward(ctx, dh):
        qx_t, sx_t, amax_x_col, qw_t, sw_t, amax_w_col, gu, w = ctx.saved_tensors
        p, op = ctx.qlinear_params, ctx.quantize_op
        if ctx.sx_t_swz is not None:
            sx_t._mt_swz = ctx.sx_t_swz
        if ctx.sw_t_swz is not None:
            sw_t._mt_swz = ctx.sw_t_swz
        dh = dh.reshape(-1, dh.shape[-1])
        M, grad_dtype = dh.shape[0], dh.dtype
        dh = cast_if_needed(dh, torch.bfloat16)
        if M == 0:
            dh = _pad_rows(dh, ctx.rows)
        # (rows that continue a ragged batch have no gradient: the kernel takes dh without them)
        qres_d = op.gated_backward(dh, gu, p.g_params, ctx.activation)
        dgrad = op.qgemm(qres_d.data, qw_t, p.mm_dgrad, p.mm_dgrad.out_dtype or grad_dtype, qres_d.scale, sw_t, None, None,
                         accumulate=False, global_amax_qx=qres_d.global_amax_row, global_amax_qw=amax_w_col,
                         qparams_x=p.g_params, qparams_w=p.w_params)
        handle = None
        if ctx.parallel_mode == "column" and ctx.tp_size > 1:
            dgrad, handle = allreduce(dgrad, ctx.tp_group, True)
        wgrad = None
        if w.requires_grad:
            accumulate = ctx.fuse_wgrad_accumulation and (ctx.is_first_microbatch is None or not ctx.is_first_microbatch)
            main_grad = w.main_grad if ctx.fuse_wgrad_accumulation else None
            # an all-reduce of dgrad is in flight: leave it SMs to run on
            with _sm_margin(op, _overlap_sm_margin() if handle is not None else 0):
                wgrad = op.qgemm(qres_d.data_t, qx_t, p.mm_wgrad,
                                 main_grad.dtype if main_grad is not None else (p.mm_wgrad.out_dtype or w.dtype), qres_d.scale_t,
                                 sx_t, None, out=main_grad, accumulate=accumulate, global_amax_qx=qres_d.global_amax_col,
                                 global_amax_qw=amax_x_col, qparams_x=p.g_params, qparams_w=p.x_params)
            wgrad = _QuantizedLinear.reset_wgrad_if_needed(ctx, w, wgrad)
        if handle is not None:
            handle.wait()
        return (dgrad[:M].view(ctx.x_shape), None, wgrad) + (None,) * (_NUM_FN_ARGS - 3)


def _non_quantized(x, w, activation):
    g, u = torch.nn.functional.linear(x, w).chunk(2, dim=-1)
    a = torch.nn.functional.silu(g) if activation == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    return a * u


@torch._dynamo.disable(recursive=True)
def gated_linear(x: torch.Tensor, weight: torch.Tensor, *, activation: str = "silu",
                 qlinear_params: Optional[config.QLinearParams] = None,
                 inp_meta: Optional[quantization.QuantizeInputMetaBase] = None) -> torch.Tensor:
    """Functional form of GatedLinear: act(x Wg^T) * (x Wu^T) for weight = [Wg; Wu] of shape [2F, K], quantized by
    the recipe (default: the one of QAT_PARAMS) in this call, with gradients of x and weight."""
    kernels._activation_code(activation)
    if weight.dim() != 2 or weight.shape[0] % 2 or x.shape[-1] != weight.shape[1]:
        raise kernels._lib.MtError(f"gated_linear of x {tuple(x.shape)} with a weight of shape {tuple(weight.shape)}")
    params = config.get_qlinear_params_from_env_qat_params() if qlinear_params is None else qlinear_params
    if not params.quantize:
        return _non_quantized(x, weight, activation)
    refuse_tangents("gated_linear", x, weight)
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
    args = (x, inp_meta, weight, None, activation, None, 1, None, params, x.dtype, grad, None,
            False, None)
    return _QuantizedGatedLinear.apply(*args) if grad else _QuantizedGatedLinear.forward(None, *args)


class GatedLinear(LayerLinearBaseModule):
    """h = act(x Wg^T) * (x Wu^T); `weight` is [Wg; Wu], [2 * ffn_size, in_features] (a fused gate/up `Linear`
    weight fits as it is). activation: "silu" or "gelu" (tanh form). in_features and ffn_size are multiples
    of 32. No bias. parallel_mode: None or "column" (ffn_size divided over the ranks, each rank holding its
    own [gate shard; up shard]). Other arguments as in `Linear`.

    emit_quantized (attribute, off by default): `output_meta` holds what the next layer's quantizer can
    take over for h, to be given as its `inp_meta`: the row-wise MXFP8 copy, as long as h lives (used by a forward pass
    without gradients; a training pass also needs a transposed copy and quantizes h itself), or max |h|
    under an NVFP4 recipe."""

    def __init__(self, in_features: int, ffn_size: int, activation: str = "silu", fuse_wgrad_accumulation: bool = False,
                 tp_group=None, tp_size: int = 1, get_rng_state_tracker: Optional[Callable] = None,
                 rng_tracker_name: Optional[str] = None, init_method: Optional[Callable] = None,
                 params_dtype: Optional[torch.dtype] = None, parallel_mode: Optional[str] = None,
                 device: Union[torch.device, str] = "cuda", layer_name: Optional[str] = None,
                 layer_number: Optional[int] = None, qlinear_params: Optional[config.QLinearParams] = None) -> None:
        super().__init__(tp_group, tp_size, False)
        kernels._activation_code(activation)
        if parallel_mode not in ("column", None):
            raise kernels._lib.MtError(f"GatedLinear: parallel_mode {parallel_mode!r} is not supported (None or 'column')")
        params_dtype = torch.get_default_dtype() if params_dtype is None else params_dtype
        if self.tp_size > 1 and torch.cuda.is_available():
            kernels.set_launch_overlap(False)      # as Linear does: kernels resident early would take the SMs of the exchanges
        self.in_features, self.activation, self.parallel_mode = in_features, activation, parallel_mode
        self.ffn_size = divide(ffn_size, self.tp_size) if parallel_mode == "column" else ffn_size
        if self.in_features % 32 or self.ffn_size % 32:
            raise kernels._lib.MtError(f"GatedLinear needs multiples of 32, got in_features {in_features}, ffn_size {self.ffn_size}")
        self.fuse_wgrad_accumulation = fuse_wgrad_accumulation
        self.get_rng_state_tracker, self.rng_tracker_name = get_rng_state_tracker, rng_tracker_name
        self.layer_number, self.layer_name = layer_number, layer_name
        self.qlinear_params = self.set_qlinear_params(qlinear_params=qlinear_params, layer_number=layer_number,
                                                      layer_name=layer_name)
        if is_rank_0():
            logger.info("layer %s gated linear %s uses %s", layer_number, layer_name, self.qlinear_params)
        self.emit_quantized = False
        self.output_meta: Optional[quantization.QuantizeInputMeta] = None
        self.register_parameter("weight", torch.nn.Parameter(torch.empty(2 * self.ffn_size, in_features, device=device,
                                                                         dtype=params_dtype)),
                                init_fn=init_method, get_rng_state_tracker=get_rng_state_tracker)
        self.reset_parameters(defer_init=(device == "meta"))
        self.weight_qresult_cache = quantization.QuantizeResultCache()

    def reset_parameters(self, defer_init=False):
        super().reset_parameters(defer_init=defer_init)
        if not defer_init:
            set_tensor_model_parallel_attributes(self.weight, True, 0, 1)

    @torch._dynamo.disable(recursive=True)
    def forward(self, inp: torch.Tensor, is_first_microbatch: Optional[bool] = None,
                inp_meta: Optional[quantization.QuantizeInputMetaBase] = None):
        """is_first_microbatch as in `Linear.forward`; inp_meta: `output_meta` of the layer that made inp."""
        self.set_activation_dtype(inp)
        assert self.tp_group_initialized, "TP group not initialized"
        if inp.shape[-1] != self.in_features:
            raise kernels._lib.MtError(f"input of {inp.shape[-1]} features for a layer of {self.in_features}")
        self.output_meta = None
        if not self.qlinear_params.quantize:
            if self.parallel_mode == "column" and self.tp_size > 1:
                raise kernels._lib.MtError("GatedLinear: tensor parallelism needs a quantized recipe")
            return _non_quantized(inp, self.weight, self.activation)
        refuse_tangents("GatedLinear", inp, self.weight)
        self.weight_qresult_cache.keep = bool(self.primary_weights_in_fp8)
        grad = torch.is_grad_enabled()
        out_meta = None
        if self.emit_quantized:
            self.output_meta = quantization.QuantizeInputMeta()
            copy = getattr(self.qlinear_params.quantize_op, "format_name", None) == "mxfp8"
            out_meta = (self.output_meta, copy and not grad) if not (copy and grad) else None
        args = (inp, inp_meta, self.weight, self.weight_qresult_cache, self.activation, self.tp_group, self.tp_size,
                self.parallel_mode, self.qlinear_params, self.activation_dtype, grad, is_first_microbatch,
                self.fuse_wgrad_accumulation, out_meta)
        h = _QuantizedGatedLinear.apply(*args) if grad else _QuantizedGatedLinear.forward(None, *args)
        if out_meta is not None and out_meta[0].quantized is not None:
            out_meta[0].quantized = quantization.TensorCopies(h, out_meta[0].quantized)
        return h
