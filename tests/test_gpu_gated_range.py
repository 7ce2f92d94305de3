"""GPU tests of the gated projection and its gradient at the ends of their ranges.

Tolerances count roundings: one to bf16 is off by at most 2^-8 of the value, an exponential of z by (1 + |z|) 2^-20 of
its value (two fp32 steps of z, and the function's own error). A sigmoid below 2^-126 is a multiple of 2^-149 and so
off by up to one such step on top; for |z| > 200 it is 0 or 1."""
import math

import pytest
import torch

from minitransformer_b200 import kernels as K

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF, TINY, STEP = 2.0 ** -8, 2.0 ** -133, 2.0 ** -149


def _rand(shape, seed, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)          # (a NaN is not within anything)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off: {got[bad][:4].tolist()} for {want[bad][:4].tolist()}"


def _same_copies(a, b, what):
    for n in ("data", "scale", "scale_swz", "data_t", "scale_t", "scale_t_swz"):
        x, y = getattr(a, n), getattr(b, n)
        assert (x is None) == (y is None), (what, n)
        if x is not None:
            assert x.shape == y.shape and torch.equal(x.view(torch.uint8), y.view(torch.uint8)), (what, n)


def _act64(g, act):
    """act, act', the sigmoid inside, the slope of its argument times g (what act' multiplies s (1 - s) by), its argument."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), s, g, g
    c, a = math.sqrt(2 / math.pi), 0.044715
    z = 2 * c * (g + a * g ** 3)
    s = torch.sigmoid(z)
    slope = 2 * g * c * (1 + 3 * a * g * g)
    return g * s, s + slope * s * (1 - s), s, slope, z


def _check_gradient(dh, gu, act):
    r = K.gated_backward(dh, gu, activation=act, want_dgu=True, want_amax=True)
    g, u = gu.double().split(dh.shape[1], 1)
    a, d, s, slope, z = _act64(g, act)
    D = dh.double()
    soft = (1 + z.abs().clamp(max=200)) * 2.0 ** -20     # beyond, the sigmoid is 0 or 1
    # act' = s + slope s (1 - s): the magnitudes of both terms, where the second has not vanished
    terms = s + torch.where(s * (1 - s) > 0, (d - s).abs(), torch.zeros_like(s))
    reach = torch.where(z.abs() < 200, 1 + slope.abs(), torch.ones_like(s))
    want = torch.cat([D * u * d, D * a], 1)
    tol = torch.cat([HALF * (D * u * d).abs() + soft * (D * u).abs() * terms + (D * u).abs() * reach * STEP,
                     (HALF + torch.where(z.abs() < 200, soft, torch.zeros_like(s))) * (D * a).abs() + D.abs() * (g.abs().clamp(max=200) + 1) * STEP], 1)
    _within(r.dgu, want, tol + TINY, f"dgu {act}")
    _same_copies(r.quantized, K.quantize_mxfp8(r.dgu), "gradient")
    _same_copies(K.gated_backward(dh, gu, activation=act).quantized, r.quantized, "alone")
    assert float(r.amax) == float(r.dgu.abs().max().float())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [32, 9])
def test_gated_gradient_of_huge_gates(act, rows):
    """Gates up to the largest bf16 value: the derivative is 1 or 0 there, never a NaN, with dh of 0 as well."""
    F = 64
    g = torch.tensor([s * v for v in (16.5, 1e3, 1e9, 1e13, 1.3e13, 1e15, 1e19, 3e19, 1e30, 3.3e38) for s in (1, -1)], device="cuda").to(BF)
    gu, dh = _rand((rows, 2 * F), 1), _rand((rows, F), 2, 1e-2)
    gu[1, :20], gu[4, 30:50], gu[rows - 1, 44:64] = g, g, g
    dh[4, 30:50] = 0
    _check_gradient(dh, gu, act)
    r = K.gated_backward(dh, gu, activation=act, want_dgu=True)
    assert not bool(r.dgu[4, 30:50].any()) and not bool(r.dgu[4, F + 30:F + 50].any())


def _gates(x0, w0, up):
    """Operands whose gates are exactly x0[i] * w0[j] and whose second projection is `up`: one non-zero column each, in
    blocks of their own (x0, w0 and up on the E4M3 grid up to powers of two). Features beyond w0 have a gate of zero; with
    many rows there are enough of them for the kernel of 256-row pairs."""
    M, F, Kd = len(x0), 32 if len(x0) < 256 else 4096, 64
    x, w = torch.zeros(M, Kd, dtype=BF, device="cuda"), torch.zeros(2 * F, Kd, dtype=BF, device="cuda")
    x[:, 0], x[:, 32] = torch.tensor(x0, device="cuda").to(BF), 1.0
    w[:len(w0), 0], w[F:, 32] = torch.tensor(w0, device="cuda").to(BF), up
    q = [K.quantize_mxfp8(t, return_transpose=False) for t in (x, w)]
    g = x[:, :1].double() * w[None, :F, 0].double()
    return q, g, F


def _check_projection(x0, w0, up, act, M):
    (qx, qw), g, F = _gates((x0 * M)[:M], w0, up)
    r = K.gemm_gated_mxfp8(qx.data, qx.scale_swz, qw.data, qw.scale_swz, activation=act, sb_lin=qw.scale, want_gu=True,
                           quantize_h=True, want_amax=True)
    assert torch.equal(r.gu[:, :F].double(), g.to(BF).double()) and bool((r.gu[:, F:].double() == up).all())
    a, d, s, slope, z = _act64(g, act)
    soft = torch.where(z.abs() < 200, (1 + z.abs()) * 2.0 ** -20, torch.zeros_like(z))
    want = a * up
    _within(r.h, want, (HALF + soft) * want.abs() + (g.abs().clamp(max=200) + 1) * abs(up) * STEP + TINY, f"h {act}")
    _same_copies(r.quantized, K.quantize_mxfp8(r.h, return_transpose=False), "projection")
    assert float(r.amax) == float(r.h.abs().max().float())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M", [12, 300])
def test_gated_projection_of_huge_gates(act, M):
    x0 = [s * 2.0 ** p for p in (0, 20, 44, 50, 63) for s in (1.0, -1.75)]
    _check_projection(x0, [2.0 ** p for p in (0, 3, 20, 40, 60, 62)], 0.5, act, M)


@pytest.mark.parametrize("act,values", [("silu", [80.0, 88.0, 96.0, 104.0]), ("gelu", [7.0, 9.0, 10.0, 11.0])])
@pytest.mark.parametrize("up", [1.5, 2.0 ** 40])
@pytest.mark.parametrize("M", [8, 300])
def test_gated_projection_where_the_sigmoid_is_subnormal(act, values, up, M):
    _check_projection([-v for v in values] + values, [1.0, 1.125, 1.25, 1.5, 0.875], up, act, M)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 40])
def test_gated_gradient_where_the_sigmoid_is_subnormal(act, scale):
    """Gates whose sigmoid lies below the smallest normal fp32 value, and those at the root of act'."""
    g = {"silu": [-85, -87, -87.5, -88, -88.5, -89, -90, -92, -96, -100, -103, -104, -110, -200, -1.28125],
         "gelu": [-9.5, -9.9375, -10, -10.0625, -10.125, -10.25, -10.5, -10.75, -11, -12, -14, -20, -0.75390625]}[act]
    gu, dh = _rand((64, 128), 1), _rand((64, 64), 2)
    gu[7, :len(g)] = torch.tensor(g, device="cuda").to(BF)
    gu[:, 64:] = 1.5
    dh[7] = scale
    _check_gradient(dh, gu, act)


def test_infinities_and_nan_reach_the_projection():
    """NaN codes and infinite projections: h is NaN or infinite where the formula is, its copies are the quantize kernel's."""
    for M, F in ((40, 96), (300, 4096)):
        for act in ("silu", "gelu"):
            x, w = _rand((M, 64), 1), _rand((2 * F, 64), 2, 0.05)
            qx, qw = (K.quantize_mxfp8(t, return_transpose=False) for t in (x, w))
            clean = K.gemm_gated_mxfp8(qx.data, qx.scale_swz, qw.data, qw.scale_swz, activation=act, sb_lin=qw.scale, quantize_h=True)
            qx.data[3, 5] = 0x7F                                   # a NaN among the inputs
            qw.data[9, 7] = 0x7F                                   # ... and in a gate's weights
            r = K.gemm_gated_mxfp8(qx.data, qx.scale_swz, qw.data, qw.scale_swz, activation=act, sb_lin=qw.scale, quantize_h=True, want_amax=True)
            bad = torch.isnan(r.h)
            want = torch.zeros_like(bad)
            want[3], want[:, 9] = True, True
            assert torch.equal(bad, want) and torch.equal(r.h[~bad], clean.h[~bad])
            _same_copies(r.quantized, K.quantize_mxfp8(r.h, return_transpose=False), "nan")
            assert float(r.amax) == float(r.h[~bad].abs().max().float())
    # infinite projections: 2^100 * 2^100, and a second projection of both signs
    for M in (8, 300):
        x0 = ([2.0 ** 100, -2.0 ** 100, 1.0, 0.0] * M)[:M]
        for act in ("silu", "gelu"):
            (qx, qw), g, F = _gates(x0, [2.0 ** 100, 1.0, -2.0 ** 100], 2.0)
            r = K.gemm_gated_mxfp8(qx.data, qx.scale_swz, qw.data, qw.scale_swz, activation=act, sb_lin=qw.scale, want_gu=True, quantize_h=True)
            assert bool((r.h[0::4, 0] == float("inf")).all()) and bool((r.h[1::4, 2] == float("inf")).all())
            assert bool(torch.isnan(r.h[0::4, 2]).all())           # -inf * 0, as the formula has it
            assert bool((r.h[3::4] == 0).all())
            _same_copies(r.quantized, K.quantize_mxfp8(r.h, return_transpose=False), "inf")


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_infinities_and_nan_in_the_gradient(act):
    gu, dh = _rand((96, 256), 2), _rand((96, 128), 3)
    gu[1, 3], gu[40, 128 + 5], dh[70, 9] = float("nan"), float("inf"), float("nan")
    r = K.gated_backward(dh, gu, activation=act, want_dgu=True)
    bad = ~torch.isfinite(r.dgu)
    assert bool(bad[1, 3]) and bool(bad[1, 131]) and bool(bad[40, 5]) and bool(bad[70, 9]) and bool(bad[70, 137]) and int(bad.sum()) == 5
    _same_copies(r.quantized, K.quantize_mxfp8(r.dgu), "inf")
