"""GPU tests of the norm and the gated projection against their formulas in 64 bits, and of what they share with
the library's other kernels bit for bit (MXFP8 copies).

Tolerances count roundings: one rounding to bf16 is off by at most 2^-8 of the value; fp32 sums of n terms by
n 2^-24 of the sum of their magnitudes; an exponential e^-z of an argument that is itself rounded by about
(1 + |z|) 2^-20 of its value (two fp32 steps of z, and the function's own error, which grows with |z|)."""
import math

import pytest
import torch

from minitransformer_b200 import _lib, kernels as K
from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear, gated_linear
from minitransformer_b200.module.linear import Linear
from minitransformer_b200.module.rmsnorm import RMSNorm

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = 2.0 ** -8            # one rounding to bf16
TINY = 2.0 ** -133          # smallest bf16 step
MXFP8 = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL)


def _rand(shape, seed, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _within(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() - tol).max()):.3g} over"


def _same_copies(a, b, what):
    for n in ("data", "scale", "scale_swz", "data_t", "scale_t", "scale_t_swz"):
        x, y = getattr(a, n), getattr(b, n)
        assert (x is None) == (y is None), (what, n)
        if x is not None:
            same = x.shape == y.shape and torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            assert same, (what, n)


# ---------------------------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------------------------
def _check_norm(x, gamma, r, eps, transpose, want_y=True):
    res = K.rmsnorm(x, gamma, eps, residual=r, return_transpose=transpose, want_y=want_y, want_amax=True)
    if r is None:
        assert res.h.data_ptr() == x.data_ptr() or not x.is_contiguous()
    else:
        s = x.double() + r.double()
        _within(res.h, s, (HALF + 2.0 ** -23) * s.abs() + TINY, "h")
    h = res.h.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    # sums of positive terms: at most 8 * 4 in a row and 10 in the tree, half of it after the root, then 4 roundings
    _within(res.rstd, rstd, 30 * 2.0 ** -24 * rstd, "rstd")
    y = h * rstd[:, None] * gamma.double()
    plain = K.rmsnorm(x, gamma, eps, residual=r, quantize=False)
    _within(plain.y, y, (HALF + 34 * 2.0 ** -24) * y.abs() + TINY, "y")
    if want_y:
        assert torch.equal(res.y, plain.y)
    else:
        assert res.y is None
    _same_copies(res.quantized, K.quantize_mxfp8(plain.y, return_transpose=transpose), "norm")
    assert float(res.amax) == float(plain.y.abs().max().float()) if y.numel() else True
    return res


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (3, 64), (31, 1056), (33, 96), (128, 256), (129, 2080), (200, 8192),
                                       (64, 8224), (37, 16384), (5, 32768)])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("transpose", [True, False])
def test_norm_matches_formula(rows, cols, residual, transpose):
    x, r = _rand((rows, cols), 1, 2.0), _rand((rows, cols), 2) if residual else None
    _check_norm(x, _rand((cols,), 3) + 1, r, 1e-5, transpose, want_y=not transpose)


@pytest.mark.parametrize("transpose", [True, False])
def test_norm_edge_values(transpose):
    """Rows of zeros, of one huge element, of subnormals, of equal values; an fp32 gamma with zeros in it."""
    x = _rand((64, 512), 4)
    x[3] = 0
    x[5] = 0
    x[5, 17] = 1e4
    x[7] = 1e-38
    x[9] = 2.0
    x[11, 32:64] = 0
    gamma = torch.linspace(-2, 2, 512, device="cuda")
    gamma[128:160] = 0
    _check_norm(x, gamma, None, 1e-6, transpose)
    _check_norm(x, gamma, -x, 1e-6, transpose)          # h is zero everywhere


def test_norm_strided_rows_and_copies_of_odd_layouts():
    wide = _rand((40, 3 * 256), 5)
    gamma = _rand((256,), 6)
    for view in (wide[:, 256:512], wide[::2, 8:264], wide[:, 4:260], _rand((256, 40), 7).t()):
        r = _rand(view.shape, 8)
        a = K.rmsnorm(view, gamma, residual=r)
        b = K.rmsnorm(view.contiguous(), gamma, residual=r)
        assert torch.equal(a.y, b.y) and torch.equal(a.h, b.h)
        _same_copies(a.quantized, b.quantized, "strided")
        dy = _rand(view.shape, 9)
        ga = K.rmsnorm_backward(dy, view, gamma, b.rstd, dresidual=view)
        gb = K.rmsnorm_backward(dy, view.contiguous(), gamma, b.rstd, dresidual=view.contiguous())
        assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1], gb[1])
    one = _rand((3, 264), 10)[1:2, 4:260]                # a single row off a 16-byte address
    assert torch.equal(K.rmsnorm(one, gamma).y, K.rmsnorm(one.clone(), gamma).y)


def test_norm_of_no_rows():
    r = K.rmsnorm(torch.empty(0, 64, dtype=BF, device="cuda"), _rand((64,), 1))
    assert r.y.shape == (0, 64) and r.quantized.data.shape == (0, 64) and r.quantized.data_t.shape == (64, 0)
    dx, dg = K.rmsnorm_backward(r.y, r.h, _rand((64,), 1), r.rstd)
    assert dx.shape == (0, 64) and not bool(dg.any())


@pytest.mark.parametrize("rows,cols", [(1, 32), (2, 4096), (31, 1056), (300, 96), (1021, 2080), (640, 8192), (70, 16384), (9, 32768)])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("gamma_dtype", [BF, F32])
def test_norm_gradient_matches_formula(rows, cols, residual, gamma_dtype):
    h, gamma, dy = _rand((rows, cols), 1, 2.0), _rand((cols,), 2, dtype=gamma_dtype) + 1, _rand((rows, cols), 3, 0.1)
    dres = _rand((rows, cols), 4, 0.1) if residual else None
    rstd = K.rmsnorm(h, gamma, 1e-5, quantize=False).rstd
    dx, dg = K.rmsnorm_backward(dy, h, gamma, rstd, dresidual=dres)
    H, D, G, R = h.double(), dy.double(), gamma.double(), rstd.double()[:, None]
    a = D * G
    dot = (a * H).sum(1, keepdim=True)
    want = R * a - R ** 3 * H * dot / cols + (dres.double() if residual else 0)
    mag = R * a.abs() + R ** 3 * H.abs() * (a * H).abs().sum(1, keepdim=True) / cols + (dres.double().abs() if residual else 0)
    # the dot: 8 * 4 additions in a row, 10 in the tree, a product before each; then a few roundings
    _within(dx, want, HALF * want.abs() + 60 * 2.0 ** -24 * mag + TINY, "dx")
    terms = D * H * R
    n = math.ceil(rows / 148) + 148 * 2 / 8 + 16          # in a CTA, over the CTAs, in the last step
    _within(dg, terms.sum(0), (n + 3) * 2.0 ** -24 * terms.abs().sum(0), "dgamma")
    again = K.rmsnorm_backward(dy, h, gamma, rstd, dresidual=dres)
    assert torch.equal(dx, again[0]) and torch.equal(dg, again[1])


def test_norm_gradient_against_differences():
    """The directional derivative of sum(dy * y(x, r, gamma)) in 64 bits against the kernel's gradients."""
    x, r, gamma, dy, dh = (_rand(s, i, 1.0) for i, s in enumerate([(24, 160), (24, 160), (160,), (24, 160), (24, 160)]))
    m = RMSNorm(160, params_dtype=BF)
    with torch.no_grad():
        m.weight.copy_(gamma)
    xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
    y, h = m(xs, rs)
    torch.autograd.backward([y, h], [dy, dh])
    X, G, D, DH = h.detach().double(), gamma.double(), dy.double(), dh.double()      # the gradient is taken at the rounded sum

    def f(X, G):
        return (D * X / torch.sqrt((X * X).mean(1, keepdim=True) + m.eps) * G).sum() + (DH * X).sum()

    for seed in range(3):
        vx, vg = _rand((24, 160), 50 + seed, dtype=F64), _rand((160,), 60 + seed, dtype=F64)
        step = 1e-5
        num = (f(X + step * vx, G + step * vg) - f(X - step * vx, G - step * vg)) / (2 * step)
        ana = (xs.grad.double() * vx).sum() + (m.weight.grad.double() * vg).sum()
        # gradients are rounded to bf16: an error of at most 2^-8 of each term
        tol = HALF * ((xs.grad.double() * vx).abs().sum() + (m.weight.grad.double() * vg).abs().sum())
        assert abs(float(num - ana)) <= float(tol) + 1e-6 * abs(float(num))
    assert torch.equal(xs.grad, rs.grad)
    # the residual stream alone, and the norm alone
    xs.grad = rs.grad = None
    m(xs, rs)[1].backward(dh)
    assert torch.equal(xs.grad, dh) and torch.equal(rs.grad, dh)
    xs.grad = None
    m(xs).backward(dy)
    assert xs.grad.shape == x.shape


# ---------------------------------------------------------------------------------------------
# gated projection
# ---------------------------------------------------------------------------------------------
def _act64(g, act):
    if act == "silu":
        s, z = torch.sigmoid(g), g
        return g * s, s * (1 + g * (1 - s)), s, z
    c, a = math.sqrt(2 / math.pi), 0.044715
    z = 2 * c * (g + a * g ** 3)
    s = torch.sigmoid(z)
    return g * s, s + 2 * g * s * (1 - s) * c * (1 + 3 * a * g * g), s, z


def _operands(M, F, Kd, fmt, seed):
    x, w = _rand((M, Kd), seed), _rand((2 * F, Kd), seed + 1, 0.05)
    if fmt == "mxfp8":
        q = [K.quantize_mxfp8(t, return_transpose=False) for t in (x, w)]
        vals = [v.data.view(torch.float8_e4m3fn).double() * (2.0 ** (v.scale.double() - 127)).repeat_interleave(32, 1) for v in q]
    else:
        q = [K.quantize_nvfp4(t, return_transpose=False) for t in (x, w)]
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=F64, device="cuda")
        vals = []
        for v in q:
            n = torch.stack([v.data & 15, v.data >> 4], 2).flatten(1).long()
            e = grid[n % 8] * (1 - 2 * (n // 8)).double()
            vals.append(e * v.scale.view(torch.float8_e4m3fn).double().repeat_interleave(16, 1) * v.amax_row.double() / 2688)
    return q, vals


def _run_gated(q, fmt, act, **want):
    (x, w) = q
    if fmt == "mxfp8":
        return K.gemm_gated_mxfp8(x.data, x.scale_swz, w.data, w.scale_swz, activation=act, sb_lin=w.scale, **want)
    return K.gemm_gated_nvfp4(x.data, x.scale_swz, x.amax_row, w.data, w.scale_swz, w.amax_row, activation=act, sb_lin=w.scale, **want)


@pytest.mark.parametrize("M,F,Kd", [(1, 32, 32), (1, 128, 256), (3, 224, 96), (32, 256, 1024), (33, 160, 160), (65, 384, 544),
                                    (128, 1376, 512), (129, 128, 64), (200, 96, 288), (256, 512, 1024), (300, 1376, 736), (1000, 768, 2048)])
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_projection_matches_formula(M, F, Kd, fmt, act):
    q, (x, w) = _operands(M, F, Kd, fmt, 7)
    r = _run_gated(q, fmt, act, want_gu=True, quantize_h=True, want_amax=True)
    gu, mag = x @ w.t(), x.abs() @ w.abs().t()
    acc = (Kd / 32 + 8) * 2.0 ** -22 * mag              # additions of 32 products at a time, two bits short of fp32
    _within(r.gu, gu, HALF * gu.abs() + acc + TINY, "gu")
    g, u = gu.split(F, 1)
    ag, au = acc.split(F, 1)
    a, d, s, z = _act64(g, act)
    tol = HALF * (a * u).abs() + 1.13 * ag * u.abs() + a.abs() * au + 1.13 * ag * au + (1 + z.abs()) * 2.0 ** -20 * (a * u).abs()
    _within(r.h, a * u, tol + TINY, "h")
    _same_copies(r.quantized, K.quantize_mxfp8(r.h, return_transpose=False), "gated")
    assert float(r.amax) == float(r.h.abs().max().float())
    # every output alone is what it is together with the others
    assert torch.equal(_run_gated(q, fmt, act).h, r.h)
    assert torch.equal(_run_gated(q, fmt, act, want_h=False, want_gu=True).gu, r.gu)
    _same_copies(_run_gated(q, fmt, act, want_h=False, quantize_h=True).quantized, r.quantized, "alone")
    assert K.read_device_status() == 0


@pytest.mark.parametrize("M,F,Kd", [(127, 160, 96), (191, 224, 64), (193, 1376, 96), (449, 32, 32), (640, 1792, 544), (2000, 416, 160),
                                    (90, 9600, 64), (100, 10016, 96), (193, 8192, 64), (700, 2080, 128), (1601, 800, 96)])
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
def test_gated_projection_on_both_sides_of_one_wave(M, F, Kd, fmt):
    """64-token blocks as long as one wave holds them, whole columns of tokens or 256-row pairs beyond."""
    test_gated_projection_matches_formula(M, F, Kd, fmt, "silu")


def test_gated_projection_equals_the_plain_gemm():
    """The projections are those of the library's GEMM, rounded once."""
    for M in (40, 300):
        q, _ = _operands(M, 384, 640, "mxfp8", 3)
        gu = K.gemm_mxfp8(q[0].data, q[0].scale_swz, q[1].data, q[1].scale_swz, out_dtype=torch.float32)
        got = _run_gated(q, "mxfp8", "silu", want_h=False, want_gu=True).gu
        assert float((got.float() - gu).norm() / gu.norm()) <= 2.0 ** -8
        assert float((got.float() - gu.to(BF).float()).norm() / gu.norm()) <= 1e-4


def test_gated_projection_of_empty_and_extreme_inputs():
    q, _ = _operands(4, 64, 64, "mxfp8", 5)
    empty = K.quantize_mxfp8(torch.empty(0, 64, dtype=BF, device="cuda"), return_transpose=False)
    r = _run_gated((empty, q[1]), "mxfp8", "silu", want_gu=True, quantize_h=True)
    assert r.h.shape == (0, 64) and r.gu.shape == (0, 128)
    for act in ("silu", "gelu"):
        # projections of +-1e5 and zero: the activation saturates without a NaN
        x = torch.zeros(3, 64, dtype=BF, device="cuda")
        x[0], x[1] = 50.0, -50.0
        w = torch.full((128, 64), 32.0, dtype=BF, device="cuda")
        qq = [K.quantize_mxfp8(t, return_transpose=False) for t in (x, w)]
        h = _run_gated(qq, "mxfp8", act, quantize_h=True).h.float()
        v = float(qq[0].data[0, :1].view(torch.float8_e4m3fn).float()) * 2.0 ** (int(qq[0].scale[0, 0]) - 127) * 64 * 32
        assert torch.isfinite(h).all() and bool((h[1:] == 0).all())
        assert abs(float(h[0, 0]) / (v * v) - 1) <= HALF + 1e-5


@pytest.mark.parametrize("rows,F", [(1, 32), (2, 64), (31, 96), (32, 128), (33, 1376), (127, 160), (128, 256), (130, 4096), (1021, 352)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_gradient_matches_formula(rows, F, act):
    gu, dh = _rand((rows, 2 * F), 1, 2.0), _rand((rows, F), 2, 1e-2)
    gu[0, 0], gu[0, F] = -200.0, 3.0
    gu[-1, 1] = 200.0
    r = K.gated_backward(dh, gu, activation=act, want_dgu=True, want_amax=True)
    g, u = gu.double().split(F, 1)
    a, d, s, z = _act64(g, act)
    D = dh.double()
    soft = (1 + z.abs()) * 2.0 ** -20
    slope = (s + (d - s).abs())                          # magnitudes of the two terms of act'
    want = torch.cat([D * u * d, D * a], 1)
    tol = torch.cat([HALF * (D * u * d).abs() + soft * (D * u).abs() * slope, (HALF + soft) * (D * a).abs()], 1)
    _within(r.dgu, want, tol + TINY, "dgu")
    _same_copies(r.quantized, K.quantize_mxfp8(r.dgu), "gradient")
    assert float(r.amax) == float(r.dgu.abs().max().float())
    if rows > 1:     # dh with fewer rows: as with zeros in the rest
        n = rows // 2 + 1
        part = K.gated_backward(dh[:n], gu, activation=act, want_dgu=True)
        full = K.gated_backward(torch.cat([dh[:n], torch.zeros_like(dh[n:])]), gu, activation=act, want_dgu=True)
        assert torch.equal(part.dgu, full.dgu) and not bool(part.dgu[n:].any())
        _same_copies(part.quantized, full.quantized, "fewer rows")
    alone = K.gated_backward(dh, gu, activation=act)
    assert alone.dgu is None and alone.amax is None
    _same_copies(alone.quantized, r.quantized, "alone")


def test_gated_gradient_against_differences():
    for act in ("silu", "gelu"):
        gu, dh, v = _rand((16, 128), 1, 1.5), _rand((16, 64), 2), _rand((16, 128), 3, dtype=F64)
        got = K.gated_backward(dh, gu, activation=act, quantize=False, want_dgu=True).dgu.double()

        def f(t):
            return (dh.double() * _act64(t[:, :64], act)[0] * t[:, 64:]).sum()

        step = 1e-5
        num = (f(gu.double() + step * v) - f(gu.double() - step * v)) / (2 * step)
        assert abs(float(num - (got * v).sum())) <= HALF * float((got * v).abs().sum()) + 1e-6


# ---------------------------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------------------------
def _values(q, s):
    return q.view(torch.float8_e4m3fn).double() * torch.repeat_interleave(2.0 ** (s.double() - 127), 32, 1)[:, :q.shape[1]]


@pytest.mark.parametrize("shape", [(64, 256, 128), (200, 96, 1376), (33, 512, 160), (1, 64, 32), (512, 1024, 768)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_linear_forward_and_backward(shape, act):
    """Against the same quantized products in 64 bits, the projections taken as the kernel saves them."""
    M, Kd, F = shape
    x, w, dh = _rand((M, Kd), 1), _rand((2 * F, Kd), 2, 0.05), _rand((M, F), 3, 1e-2)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    h = gated_linear(xs, ws, activation=act, qlinear_params=MXFP8)
    dx, dw = torch.autograd.grad(h, (xs, ws), dh)
    qx, qw = K.quantize_mxfp8(torch.nn.functional.pad(x, (0, 0, 0, -M % 32))), K.quantize_mxfp8(w)
    r = K.gemm_gated_mxfp8(qx.data, qx.scale_swz, qw.data, qw.scale_swz, activation=act, sb_lin=qw.scale, want_gu=True)
    assert torch.equal(h, r.h[:M])
    dgu = K.gated_backward(torch.nn.functional.pad(dh, (0, 0, 0, -M % 32)), r.gu, activation=act).quantized
    want = _values(dgu.data, dgu.scale) @ _values(qw.data_t, qw.scale_t).t()
    mag = _values(dgu.data, dgu.scale).abs() @ _values(qw.data_t, qw.scale_t).abs().t()
    _within(dx, want[:M], HALF * want[:M].abs() + (2 * F / 32 + 8) * 2.0 ** -22 * mag[:M] + TINY, "dx")
    want = _values(dgu.data_t, dgu.scale_t) @ _values(qx.data_t, qx.scale_t).t()
    mag = _values(dgu.data_t, dgu.scale_t).abs() @ _values(qx.data_t, qx.scale_t).abs().t()
    _within(dw, want, HALF * want.abs() + (M / 32 + 9) * 2.0 ** -22 * mag + TINY, "dw")
    # without gradients nothing is padded and nothing saved; the result is the same
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w, activation=act, qlinear_params=MXFP8), h)


@pytest.mark.parametrize("recipe", [config.QuantizeRecipe.FP4_SUB_CHANNEL, config.QuantizeRecipe.FP4_SUB_CHANNEL_NO_RHT])
def test_gated_linear_nvfp4_equals_its_parts(recipe):
    p = config.get_qlinear_params_from_predefined(recipe)
    M, Kd, F = 200, 256, 384
    x, w, dh = _rand((M, Kd), 1).requires_grad_(), _rand((2 * F, Kd), 2, 0.05).requires_grad_(), _rand((M, F), 3, 1e-2)
    h = gated_linear(x, w, qlinear_params=p)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    # the same with Linear for the projections and torch for the rest: only roundings in between differ
    lin = Linear(Kd, 2 * F, bias=False, params_dtype=BF, qlinear_params=p)
    with torch.no_grad():
        lin.weight.copy_(w)
    x2 = torch.nn.functional.pad(x.detach(), (0, 0, 0, -M % 32)).requires_grad_()
    g, u = lin(x2).chunk(2, -1)
    h2 = torch.nn.functional.silu(g) * u
    h2.backward(torch.nn.functional.pad(dh, (0, 0, 0, -M % 32)))
    rel = lambda a, b: float(((a.float() - b.float()).norm() / b.float().norm()).detach())  # noqa: E731
    # h: four roundings of the torch path (g, u, silu, product) against one; gradients: of every 2^-8 that the bf16
    # gradient differs by, 4-bit codes (half a step is up to 1/4 of the value) can turn some over
    assert rel(h, h2[:M]) <= 4 * HALF
    assert rel(dx, x2.grad[:M]) <= 0.1 and rel(dw, lin.weight.grad) <= 0.1


def test_block_of_norm_gated_projection_and_linear():
    """RMSNorm -> GatedLinear -> Linear as a block uses them: what the layers hand each other (copies made by the
    norm, by the gated projection) changes nothing, forward and backward."""
    H, F, M = 256, 384, 160
    norm = RMSNorm(H, params_dtype=BF, qlinear_params=MXFP8)
    fc1 = GatedLinear(H, F, params_dtype=BF, qlinear_params=MXFP8)
    fc2 = Linear(F, H, bias=False, params_dtype=BF, qlinear_params=MXFP8)
    x, r, dy = _rand((M, H), 1), _rand((M, H), 2), _rand((M, H), 3, 1e-2)

    def block(fused):
        norm.emit_quantized = fc1.emit_quantized = fused
        y, h = norm(xs, rs)
        a = fc1(y, inp_meta=norm.output_meta)
        return h + fc2(a, inp_meta=fc1.output_meta)

    grads = []
    for fused in (False, True):
        for p in (*norm.parameters(), *fc1.parameters(), *fc2.parameters()):
            p.grad = None
        xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
        out = block(fused)
        out.backward(dy)
        with torch.no_grad():
            served = block(fused)
        if fused:
            assert norm.output_meta.quantized is not None and fc1.output_meta.quantized is not None
        assert torch.equal(served, out)
        grads.append([out, xs.grad, rs.grad, norm.weight.grad, fc1.weight.grad, fc2.weight.grad])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_gated_linear_weight_cache_and_main_grad():
    lin = GatedLinear(128, 256, params_dtype=BF, fuse_wgrad_accumulation=True, qlinear_params=MXFP8)
    lin.weight.main_grad = torch.zeros(512, 128, device="cuda")
    x, dh = _rand((64, 128), 1), _rand((64, 256), 2, 1e-2)
    with torch.no_grad():
        lin(x, is_first_microbatch=True)                     # fills the cache without a transposed copy
    for first in (True, False):
        lin(x.clone().requires_grad_(), is_first_microbatch=first).backward(dh)
    assert lin.weight.grad is None
    ref = GatedLinear(128, 256, params_dtype=BF, qlinear_params=MXFP8)
    with torch.no_grad():
        ref.weight.copy_(lin.weight)
    ref(x.clone().requires_grad_()).backward(dh)
    got = lin.weight.main_grad / 2
    _within(ref.weight.grad, got.double(), HALF * got.double().abs() + 2.0 ** -22 * got.double().abs() + TINY, "main_grad")
    kept = lin(x)
    lin.keep_quantized_weights()
    with torch.no_grad():
        lin.weight.zero_()
    assert torch.equal(lin(x), kept)
    lin.refresh_quantized_weights()
    assert not bool(lin(x).any())


def test_fp32_gamma_and_bf16_recipe():
    plain = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.NON_QUANTIZE)
    norm = RMSNorm(64, params_dtype=torch.float32, qlinear_params=plain)
    norm.emit_quantized = True
    x = _rand((2, 5, 64), 1).requires_grad_()
    lin = GatedLinear(64, 96, activation="gelu", params_dtype=BF, qlinear_params=plain)
    y = lin(norm(x), inp_meta=norm.output_meta)
    assert y.shape == (2, 5, 96) and norm.output_meta is None
    y.sum().backward()
    assert norm.weight.grad.dtype == torch.float32 and x.grad.shape == x.shape


# ---------------------------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------------------------
def test_other_stream_and_two_graphs():
    """A training pass captured twice (two graphs, memory of their own) and replayed in turn on new inputs."""
    norm = RMSNorm(128, params_dtype=BF, qlinear_params=MXFP8)
    norm.emit_quantized = True
    fc1 = GatedLinear(128, 160, params_dtype=BF, qlinear_params=MXFP8)
    data = [[_rand((96, 128), 10 * i + j) for j in range(2)] + [_rand((96, 160), 10 * i + 5, 1e-2)] for i in range(3)]

    def step(x, r, dh):
        y, h = norm(x, r)
        a = fc1(y, inp_meta=norm.output_meta)
        return [a, h, *torch.autograd.grad(a, (x, r, norm.weight, fc1.weight), dh)]

    # (results without their graphs: torch cannot capture a backward pass while an eager graph of the same
    # parameters lives, whatever its layers are)
    eager = [[t.detach().clone() for t in step(x.clone().requires_grad_(), r.clone().requires_grad_(), dh)] for x, r, dh in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for (x, r, dh), want in zip(data, eager):
            got = step(x.clone().requires_grad_(), r.clone().requires_grad_(), dh)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            del got
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        static = [data[0][0].clone().requires_grad_(), data[0][1].clone().requires_grad_(), data[0][2].clone()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*static)
        graphs.append((g, static, out))
    for (x, r, dh), want in zip(data, eager):
        for g, static, out in graphs:
            with torch.no_grad():
                for s, t in zip(static, (x, r, dh)):
                    s.copy_(t)
            g.replay()
        for g, static, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_amax_in_a_replayed_graph_starts_from_zero():
    x, gamma = _rand((32, 64), 1, 8.0), torch.ones(64, dtype=BF, device="cuda")
    gu, dh = _rand((32, 128), 2), _rand((32, 64), 3)
    K.rmsnorm(x, gamma, want_amax=True, quantize=False)
    K.gated_backward(dh, gu, quantize=False, want_dgu=True, want_amax=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = K.rmsnorm(x, gamma, want_amax=True, quantize=False)
        b = K.gated_backward(dh, gu, quantize=False, want_dgu=True, want_amax=True)
    for scale in (8.0, 0.5):
        gamma.fill_(scale)
        dh.copy_(_rand((32, 64), 4, scale))
        g.replay()
        assert float(a.amax) == float(a.y.abs().max()) and float(b.amax) == float(b.dgu.abs().max())


def test_refusals_on_the_gpu():
    x, w = _rand((4, 64), 1), _rand((64,), 2)
    bad = [lambda: K.rmsnorm(x.float(), w), lambda: K.rmsnorm(x, w[:32]), lambda: K.rmsnorm(x, w.half()),
           lambda: K.rmsnorm(x, w, residual=x[:2]), lambda: K.rmsnorm(x, w.cpu()), lambda: K.rmsnorm(x[:, :20].contiguous(), w[:20]),
           lambda: K.rmsnorm(x[:, :24].contiguous(), w[:24]), lambda: K.rmsnorm(x, w, want_y=False, quantize=False),
           lambda: K.rmsnorm(x, w, eps=-1.0), lambda: K.rmsnorm(_rand((1, 32800), 1), _rand((32800,), 1)),
           lambda: K.rmsnorm_backward(x, x, w, torch.ones(3, device="cuda")),
           lambda: K.gated_backward(x, x), lambda: K.gated_backward(x, _rand((3, 128), 1)),
           lambda: K.gated_backward(x[:0], _rand((3, 128), 1)), lambda: K.gated_backward(x, _rand((4, 128), 1), activation="tanh"),
           lambda: K.gated_backward(x[:, :48], _rand((4, 96), 1)),
           lambda: gated_linear(x, _rand((65, 64), 1), qlinear_params=MXFP8),
           lambda: gated_linear(x.float(), _rand((64, 64), 1), qlinear_params=MXFP8),
           lambda: GatedLinear(40, 64, qlinear_params=MXFP8), lambda: GatedLinear(64, 64, parallel_mode="row", qlinear_params=MXFP8),
           lambda: RMSNorm(64, params_dtype=BF)(x, x[:1])]
    for f in bad:
        with pytest.raises(_lib.MtError):
            f()
    q, _ = _operands(4, 96, 64, "mxfp8", 1)
    with pytest.raises(_lib.MtError, match="sb_lin"):
        K.gemm_gated_mxfp8(q[0].data, q[0].scale_swz, q[1].data, q[1].scale_swz)
    with pytest.raises(_lib.MtError, match="smaller than"):
        K.gemm_gated_mxfp8(q[0].data, q[0].scale_swz[:512], q[1].data, q[1].scale_swz, sb_lin=q[1].scale)
    norm = RMSNorm(64, params_dtype=BF, qlinear_params=MXFP8)
    norm.emit_quantized = True
    norm(x)
    with pytest.raises(_lib.MtError, match="copies of"):
        with torch.no_grad():
            GatedLinear(64, 64, params_dtype=BF, qlinear_params=MXFP8)(x[:2], inp_meta=norm.output_meta)
    assert K.read_device_status() == 0


@pytest.mark.parametrize("rows,cols", [(5, 96), (700, 2080), (300, 4096)])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_norm_in_place(rows, cols, transpose, into):
    """The sum in the place of x or of the residual, the gradient in the place of dres (C ABI)."""
    x, r, w, dy, d = _rand((rows, cols), 1), _rand((rows, cols), 2), _rand((cols,), 3), _rand((rows, cols), 4), _rand((rows, cols), 5)
    want = K.rmsnorm(x, w, residual=r, return_transpose=transpose)
    c = K._mxfp8_outputs(rows, cols, transpose, x.device)
    y, rstd, stream = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.cuda.current_stream().cuda_stream
    h = {"x": x, "residual": r}[into]
    ptr = K._ptr
    _lib.call("mt_rmsnorm_forward", ptr(x), cols, ptr(r), cols, ptr(w), _lib.MT_BF16, rows, cols, 1e-5, ptr(h), ptr(rstd), ptr(y),
              None, ptr(c.data), ptr(c.scale), cols // 32, ptr(c.scale_swz), ptr(c.data_t), ptr(c.scale_t), (rows + 31) // 32,
              ptr(c.scale_t_swz), stream)
    assert torch.equal(h, want.h) and torch.equal(y, want.y) and torch.equal(rstd, want.rstd)
    _same_copies(c, want.quantized, "in place")
    dx, dw = K.rmsnorm_backward(dy, h, w, rstd, dresidual=d)
    dw2 = torch.empty_like(dw)
    n = _lib.load().mt_rmsnorm_backward_workspace(rows, cols)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    _lib.call("mt_rmsnorm_backward", ptr(dy), cols, ptr(h), cols, ptr(w), _lib.MT_BF16, ptr(rstd), ptr(d), cols, rows, cols, ptr(d),
              ptr(dw2), ptr(work), n, stream)
    assert torch.equal(d, dx) and torch.equal(dw2, dw)
    assert K.read_device_status() == 0


def test_operands_that_do_not_belong_together_are_refused():
    q, _ = _operands(4, 96, 64, "mxfp8", 1)
    with pytest.raises(_lib.MtError, match="sb_lin"):      # row-major scales of a shorter weight
        K.gemm_gated_mxfp8(q[0].data, q[0].scale_swz, q[1].data, q[1].scale_swz, sb_lin=q[1].scale[:, :1])
    with pytest.raises(_lib.MtError, match="contiguous"):
        K.gemm_gated_mxfp8(q[0].data, torch.cat([q[0].scale_swz] * 2)[::2], q[1].data, q[1].scale_swz, sb_lin=q[1].scale)
    f, _ = _operands(4, 128, 64, "nvfp4", 1)
    for a, b in ((None, f[1].amax_row), (f[0].amax_row, None), (f[0].amax_row.double(), f[1].amax_row)):
        with pytest.raises(_lib.MtError, match="fp32 device scalar"):
            K.gemm_gated_nvfp4(f[0].data, f[0].scale_swz, a, f[1].data, f[1].scale_swz, b)
    x, w = _rand((4, 64), 1), _rand((64,), 2)
    a, b = K.rmsnorm(x, w), K.rmsnorm(x=x, weight=w)
    assert torch.equal(a.y, b.y) and torch.equal(a.quantized.data, b.quantized.data)


@pytest.mark.parametrize("rows,cols", [(700, 64), (1021, 2080), (640, 8192), (593, 4096), (600, 16384)])
def test_norm_of_many_rows(rows, cols):
    """Rows enough for the persistent kernels, each CTA taking several: same bits as the same rows in small batches."""
    x, r, gamma = _rand((rows, cols), 1, 2.0), _rand((rows, cols), 2), _rand((cols,), 3) + 1
    for residual in (r, None):
        for transpose in (False, True):
            res = _check_norm(x, gamma, residual, 1e-5, transpose)
        for a in range(0, rows, 250):
            part = K.rmsnorm(x[a:a + 250], gamma, 1e-5, residual=None if residual is None else r[a:a + 250], quantize=False)
            assert torch.equal(part.y, res.y[a:a + 250]) and torch.equal(part.rstd, res.rstd[a:a + 250])
    assert K.read_device_status() == 0


def test_infinities_and_nan_reach_the_copies_as_in_the_quantize_kernel():
    """Inputs with infinities and NaN: y and dgu carry them where the formula does, and the copies are the quantize
    kernel's, finite blocks untouched."""
    x = _rand((64, 256), 1)
    x[3, 5], x[40, 7] = float("inf"), float("nan")
    gamma = torch.ones(256, dtype=BF, device="cuda")
    for transpose in (True, False):
        r = K.rmsnorm(x, gamma, return_transpose=transpose)
        bad = ~torch.isfinite(r.y).all(1)
        assert bad[3] and bad[40] and int(bad.sum()) == 2
        _same_copies(r.quantized, K.quantize_mxfp8(r.y, return_transpose=transpose), "inf")
    gu, dh = _rand((64, 128), 2), _rand((64, 64), 3)
    gu[1, 64 + 3], dh[33, 9] = float("inf"), float("-inf")
    r = K.gated_backward(dh, gu, want_dgu=True)
    assert bool(torch.isinf(r.dgu[1, 3])) and bool(torch.isinf(r.dgu[33, 64 + 9])) and int((~torch.isfinite(r.dgu)).sum()) == 3
    _same_copies(r.quantized, K.quantize_mxfp8(r.dgu), "inf")


def test_gated_linear_without_tokens_and_under_autocast():
    lin = GatedLinear(64, 96, params_dtype=BF, qlinear_params=MXFP8)
    x = torch.empty(0, 64, dtype=BF, device="cuda", requires_grad=True)
    h = lin(x)
    h.sum().backward()
    assert h.shape == (0, 96) and x.grad.shape == (0, 64) and not bool(lin.weight.grad.any())
    master = GatedLinear(64, 96, params_dtype=torch.float32, qlinear_params=MXFP8)
    with torch.no_grad():
        master.weight.copy_(lin.weight)
    x = _rand((48, 64), 1, dtype=torch.float32).requires_grad_()
    with torch.autocast("cuda", dtype=BF):
        h = master(x)
    h.backward(_rand((48, 96), 2))
    xb = x.detach().to(BF).requires_grad_()
    lin.weight.grad = None
    hb = lin(xb)
    hb.backward(_rand((48, 96), 2))
    assert torch.equal(h, hb) and x.grad.dtype == torch.float32 and master.weight.grad.dtype == torch.float32
    assert torch.equal(x.grad, xb.grad.float()) and torch.equal(master.weight.grad.to(BF), lin.weight.grad)
    with pytest.raises(_lib.MtError, match="bf16"):
        with torch.autocast("cuda", dtype=torch.float16):
            master(x)


def test_results_do_not_depend_on_what_ran_before():
    """Kernels that start early wait for the one before them: chains of dependent calls, many times, same bits."""
    x, r, gamma = _rand((300, 512), 1), _rand((300, 512), 2), _rand((512,), 3) + 1
    w, dh = _rand((768, 512), 4, 0.05), _rand((300, 384), 5, 1e-2)
    qw = K.quantize_mxfp8(w)

    def chain():
        n = K.rmsnorm(x, gamma, residual=r)
        g = K.gemm_gated_mxfp8(n.quantized.data, n.quantized.scale_swz, qw.data, qw.scale_swz, want_gu=True, quantize_h=True)
        b = K.gated_backward(dh, g.gu)
        d = K.gemm_mxfp8(b.quantized.data, b.quantized.scale_swz, qw.data_t, qw.scale_t_swz)
        dx, dg = K.rmsnorm_backward(d, n.h, gamma, n.rstd, dresidual=n.h)
        return [n.y, g.h, g.quantized.data, b.quantized.data_t, dx, dg]

    first = chain()
    for _ in range(30):
        again = chain()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    before = K.set_launch_overlap(False)
    try:
        assert all(torch.equal(a, b) for a, b in zip(first, chain()))
    finally:
        K.set_launch_overlap(before)
    assert K.read_device_status() == 0


@pytest.mark.parametrize("rows,cols", [(8192, 4096), (15665, 704), (15664, 2080), (6001, 8192)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_of_many_panels_repeated(rows, cols, residual):
    """Clusters that take several panels one after the other, tiles arriving while the ones before are in use."""
    x, r, gamma = _rand((rows, cols), 1, 2.0), _rand((rows, cols), 2) if residual else None, _rand((cols,), 3) + 1
    plain = K.rmsnorm(x, gamma, residual=r, quantize=False)
    copies = K.quantize_mxfp8(plain.y)
    for _ in range(12):
        res = K.rmsnorm(x, gamma, residual=r)
        assert torch.equal(res.rstd, plain.rstd) and torch.equal(res.y, plain.y) and torch.equal(res.h, plain.h)
        _same_copies(res.quantized, copies, "panels")
    assert K.read_device_status() == 0


@pytest.mark.parametrize("rows,F", [(8192, 4096), (4099, 1376), (2048, 14336)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_gradient_of_many_tiles_repeated(rows, F, act):
    gu, dh = _rand((rows, 2 * F), 1, 1.5), _rand((rows, F), 2, 1e-2)
    dgu = K.gated_backward(dh, gu, activation=act, quantize=False, want_dgu=True).dgu
    g, u = gu.double().split(F, 1)
    a, d, s, z = _act64(g, act)
    D = dh.double()
    soft, slope = (1 + z.abs()) * 2.0 ** -20, s + (d - s).abs()
    _within(dgu[:, :F], D * u * d, HALF * (D * u * d).abs() + soft * (D * u).abs() * slope + TINY, "dg")
    _within(dgu[:, F:], D * a, (HALF + soft) * (D * a).abs() + TINY, "du")
    del g, u, a, d, s, z, D, soft, slope
    copies = K.quantize_mxfp8(dgu)
    for _ in range(12):
        r = K.gated_backward(dh, gu, activation=act, want_dgu=True)
        assert torch.equal(r.dgu, dgu)
        _same_copies(r.quantized, copies, "tiles")
    assert K.read_device_status() == 0


@pytest.mark.parametrize("rows,cols", [(8192, 8192), (9001, 2080), (5000, 704)])
def test_norm_gradient_of_many_rows_repeated(rows, cols):
    h, gamma, dy, dres = _rand((rows, cols), 1, 2.0), _rand((cols,), 2) + 1, _rand((rows, cols), 3, 0.1), _rand((rows, cols), 4, 0.1)
    rstd = K.rmsnorm(h, gamma, quantize=False).rstd
    first = K.rmsnorm_backward(dy, h, gamma, rstd, dresidual=dres)
    H, R, A = h.double(), rstd.double()[:, None], dy.double() * gamma.double()
    want = R * A - R ** 3 * H * (A * H).sum(1, keepdim=True) / cols + dres.double()
    mag = R * A.abs() + R ** 3 * H.abs() * (A * H).abs().sum(1, keepdim=True) / cols + dres.double().abs()
    _within(first[0], want, HALF * want.abs() + 60 * 2.0 ** -24 * mag + TINY, "dx")
    for _ in range(12):
        again = K.rmsnorm_backward(dy, h, gamma, rstd, dresidual=dres)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    assert K.read_device_status() == 0


def test_decoder_with_fused_blocks_stays_within_quantization_noise():
    """The benchmark's decoder, small: the fused block against the same model in bf16, with the bounds that the plain
    MXFP8 decoder is held to; and close to that decoder itself, from which only roundings separate it."""
    import bench
    dims = dict(layers=2, hidden=256, heads=4, kv_heads=2, ffn=512, vocab=512)
    plain = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.NON_QUANTIZE)
    torch.manual_seed(0)
    models = [bench.build_llama_decoder(torch, dims, p, fused_block=f) for p, f in ((MXFP8, True), (MXFP8, False), (plain, False), (plain, True))]
    for m in models[1:]:
        m.load_state_dict(models[0].state_dict())
    ids, tgt = (torch.randint(0, 512, (2, 128), device="cuda") for _ in range(2))
    losses, grads = [], []
    for m in models:
        loss = m(ids, tgt)
        loss.backward()
        losses.append(loss.item())
        grads.append(torch.cat([p.grad.float().flatten() for _, p in sorted(m.named_parameters())]))
    cos = [float(torch.nn.functional.cosine_similarity(g, grads[2], dim=0)) for g in grads]
    assert all(abs(v - losses[2]) / losses[2] < 0.02 for v in losses), losses
    assert min(cos) > 0.97, cos
    assert K.read_device_status() == 0
