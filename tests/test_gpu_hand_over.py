"""GPU tests of what the norm and the gated projection hand on to the next layer: memory, who takes it, and inputs changed in between."""
import pytest
import torch

from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear
from minitransformer_b200.module.linear import Linear
from minitransformer_b200.module.rmsnorm import RMSNorm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
MXFP8 = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL)


def _rand(shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


def _stack(emit, recipe, n=4, H=256):
    layers = []
    for _ in range(n):
        norm, lin = RMSNorm(H, params_dtype=BF, qlinear_params=recipe), Linear(H, H, bias=False, params_dtype=BF, qlinear_params=recipe)
        norm.emit_quantized = emit
        layers.append((norm, lin))
    return layers


def test_copies_do_not_outlive_the_tensor_they_belong_to():
    """A stack that hands copies on holds no more memory after its forward pass, after its backward pass and between
    calls without gradients than one that does not."""
    held = {}
    for emit in (False, True):
        layers = _stack(emit, MXFP8)
        x = _rand((1024, 256), 1).requires_grad_()

        def forward():
            y = x
            for norm, lin in layers:
                y = lin(norm(y), inp_meta=norm.output_meta)
            return y

        for _ in range(2):                                  # gradients and weight copies exist from here on
            forward().sum().backward()
        for norm, _ in layers:
            norm.output_meta = None
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        out = forward()
        after_forward = torch.cuda.memory_allocated() - base
        out.sum().backward()
        del out
        after_backward = torch.cuda.memory_allocated() - base
        with torch.no_grad():
            forward()
        held[emit] = (after_forward, after_backward, torch.cuda.memory_allocated() - base)
    assert all(a <= b for a, b in zip(held[True], held[False])), held


def test_copies_of_a_changed_tensor_are_not_used():
    norm = RMSNorm(256, params_dtype=BF, qlinear_params=MXFP8)
    norm.emit_quantized = True
    lin = Linear(256, 128, bias=False, params_dtype=BF, qlinear_params=MXFP8)
    gated = GatedLinear(256, 128, params_dtype=BF, qlinear_params=MXFP8)
    x = _rand((64, 256), 1)
    with torch.no_grad():
        for layer in (lin, gated):
            y = norm(x)
            same = layer(y, inp_meta=norm.output_meta)
            assert torch.equal(same, layer(y.clone()))
            y.mul_(-3)
            assert torch.equal(layer(y, inp_meta=norm.output_meta), layer(y.clone()))
            other = _rand((64, 256), 9)
            assert torch.equal(layer(other, inp_meta=norm.output_meta), layer(other))


def test_one_norm_feeds_several_layers_from_its_copies():
    """Three projections of one norm's output take its copies: the quantize kernel runs for their weights alone."""
    from minitransformer_b200 import kernels as K
    norm = RMSNorm(256, params_dtype=BF, qlinear_params=MXFP8)
    norm.emit_quantized = True
    layers = [Linear(256, 128, bias=False, params_dtype=BF, qlinear_params=MXFP8) for _ in range(3)]
    x = _rand((2, 32, 256), 1).requires_grad_()
    y = norm(x)
    before = K.LAUNCH_COUNT
    outs = [layer(y, inp_meta=norm.output_meta) for layer in layers]
    assert K.LAUNCH_COUNT - before == 3 * 2
    for out, layer in zip(outs, layers):
        assert torch.equal(out, layer(y.detach().clone()))
    with torch.inference_mode():
        z = norm(x)
        before = K.LAUNCH_COUNT
        served = layers[0](z, inp_meta=norm.output_meta)
        assert K.LAUNCH_COUNT - before == 2 and torch.equal(served, outs[0])
