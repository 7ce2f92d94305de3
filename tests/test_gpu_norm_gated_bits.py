"""GPU tests of the norm and the gated projection: single elements and single runs, where a norm or a last run could
hide one that is off."""
import pytest
import torch

import test_gpu_norm_gated as base
from minitransformer_b200 import kernels as K
from minitransformer_b200.module import config

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
MXFP8 = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL)
_rand = base._rand


@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
@pytest.mark.parametrize("M,F,Kd", [(1, 128, 256), (40, 384, 640), (100, 384, 640), (300, 384, 640), (700, 1376, 512), (257, 256, 4096), (700, 2080, 128), (193, 8192, 64),
                                    (1601, 800, 96)])
def test_projections_are_bits_of_the_plain_gemm(fmt, M, F, Kd):
    """Blocks of tokens and 256-row pairs (the last three): [g | u] is the plain GEMM's fp32 result, rounded once."""
    x, w = _rand((M, Kd), 3), _rand((2 * F, Kd), 4, 0.05)
    if fmt == "mxfp8":
        q = [K.quantize_mxfp8(t, return_transpose=False) for t in (x, w)]
        gu = K.gemm_mxfp8(q[0].data, q[0].scale_swz, q[1].data, q[1].scale_swz, out_dtype=torch.float32)
        got = K.gemm_gated_mxfp8(q[0].data, q[0].scale_swz, q[1].data, q[1].scale_swz, sb_lin=q[1].scale, want_h=False, want_gu=True).gu
    else:
        q = [K.quantize_nvfp4(t, return_transpose=False) for t in (x, w)]
        gu = K.gemm_nvfp4(q[0].data, q[0].scale_swz, q[0].amax_row, q[1].data, q[1].scale_swz, q[1].amax_row, out_dtype=torch.float32)
        got = K.gemm_gated_nvfp4(q[0].data, q[0].scale_swz, q[0].amax_row, q[1].data, q[1].scale_swz, q[1].amax_row, sb_lin=q[1].scale,
                                 want_h=False, want_gu=True).gu
    assert torch.equal(got, gu.to(BF))


@pytest.mark.parametrize("M,F,Kd", [(193, 8192, 64), (700, 2080, 128), (1601, 800, 96)])
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
def test_gelu_in_256_row_pairs(M, F, Kd, fmt):
    base.test_gated_projection_matches_formula(M, F, Kd, fmt, "gelu")


def test_every_one_of_many_chains_gives_the_same_bits():
    """Chains of dependent calls in a row, with nothing waiting in between: each one of them is compared."""
    x, r, gamma = _rand((300, 512), 1), _rand((300, 512), 2), _rand((512,), 3) + 1
    w, dh = _rand((768, 512), 4, 0.05), _rand((300, 384), 5, 1e-2)
    qw = K.quantize_mxfp8(w)

    def chain():
        n = K.rmsnorm(x, gamma, residual=r)
        g = K.gemm_gated_mxfp8(n.quantized.data, n.quantized.scale_swz, qw.data, qw.scale_swz, want_gu=True, quantize_h=True)
        b = K.gated_backward(dh, g.gu)
        d = K.gemm_mxfp8(b.quantized.data, b.quantized.scale_swz, qw.data_t, qw.scale_t_swz)
        dx, dg = K.rmsnorm_backward(d, n.h, gamma, n.rstd, dresidual=n.h)
        return [n.y, n.h, n.rstd, n.quantized.data, n.quantized.data_t, n.quantized.scale_t, g.h, g.gu, g.quantized.data,
                b.quantized.data, b.quantized.data_t, b.quantized.scale_t_swz, dx, dg]

    first = chain()
    torch.cuda.synchronize()
    rest = [chain() for _ in range(60)]
    for i, again in enumerate(rest):
        assert all(torch.equal(a, b) for a, b in zip(first, again)), i
    assert K.read_device_status() == 0


def test_decoder_with_fused_blocks_against_the_unfused_one():
    """The benchmark's decoder, small: with the fused block it is closer to the same decoder without it than either is
    to the model in bf16."""
    import bench
    dims = dict(layers=2, hidden=256, heads=4, kv_heads=2, ffn=512, vocab=512)
    plain = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.NON_QUANTIZE)
    torch.manual_seed(0)
    models = [bench.build_llama_decoder(torch, dims, p, fused_block=f) for p, f in ((MXFP8, True), (MXFP8, False), (plain, False))]
    for m in models[1:]:
        m.load_state_dict(models[0].state_dict())
    ids, tgt = (torch.randint(0, 512, (2, 128), device="cuda") for _ in range(2))
    grads = []
    for m in models:
        m(ids, tgt).backward()
        grads.append(torch.cat([p.grad.float().flatten() for _, p in sorted(m.named_parameters())]))
    rel = lambda a, b: float((a - b).norm() / b.norm())  # noqa: E731
    # between the two lie roundings to bf16 and the codes they move, between either and the third 8-bit operands
    assert rel(grads[0], grads[1]) < rel(grads[1], grads[2]) and rel(grads[0], grads[1]) < rel(grads[0], grads[2])
    assert K.read_device_status() == 0
