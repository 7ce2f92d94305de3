"""CPU checks of the norm and gated entry points: refusals before anything reaches a GPU, and the device guard."""
import ctypes

import pytest
import torch

from minitransformer_b200 import _lib, kernels
from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear, gated_linear
from minitransformer_b200.module.rmsnorm import RMSNorm

MXFP8 = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL)


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(8192)
    yield (ctypes.addressof(buf) + 63) // 64 * 64
    del buf


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().mt_last_error_string().decode(), _lib.load().mt_last_error_string()


def test_norm_entry_points_refuse(p):
    lib = _lib.load()

    def fwd(x=p, xs=64, r=None, rs=0, g=p, gd=0, rows=2, cols=64, eps=1e-5, h=None, y=p, q=None, s=None, ss=2, swz=None,
            qt=None, st=None, sts=1):
        return lib.mt_rmsnorm_forward(x, xs, r, rs, g, gd, rows, cols, eps, h, p, y, None, q, s, ss, swz, qt, st, sts, None, None)

    _refused(fwd(cols=12, xs=16), "multiple of 8")
    _refused(fwd(cols=0), "within")
    _refused(fwd(cols=40000, xs=40000), "within")
    _refused(fwd(rows=-1), "within")
    _refused(fwd(gd=7), "dtype")
    _refused(fwd(eps=-1.0), "eps")
    _refused(fwd(x=None), "null")
    _refused(fwd(g=None), "null")
    _refused(fwd(xs=60), "aligned rows")
    _refused(fwd(xs=68), "aligned rows")
    _refused(fwd(x=p + 2), "aligned rows")
    _refused(fwd(r=p, rs=32, h=p), "residual needs")
    _refused(fwd(r=p, rs=64), "output for the sum")
    _refused(fwd(h=p), "no sum")
    _refused(fwd(y=p + 4), "16-byte")
    _refused(fwd(cols=40, xs=40, q=p, s=p), "multiple of 32")
    _refused(fwd(q=p), "need s")
    _refused(fwd(q=p, s=p, ss=1), "need s")
    _refused(fwd(q=p, s=p, qt=p), "need s_t")
    _refused(fwd(q=p, s=p, qt=p, st=p, sts=0), "need s_t")
    _refused(fwd(q=p, s=p, st=p), "without transposed codes")
    _refused(fwd(qt=p, st=p), "without codes")
    assert fwd(cols=8224, xs=8224, q=p, s=p, ss=257, qt=p, st=p) == -2
    _refused(fwd(q=p + 8, s=p), "16-byte")
    _refused(fwd(s=p), "without codes")
    assert fwd(rows=0, x=None) == 0                 # nothing to do

    def bwd(dy=p, dys=64, h=p, hs=64, g=p, gd=0, rstd=p, dres=None, drs=0, rows=2, cols=64, dx=p, dg=p, ws=p, wb=1 << 20):
        return lib.mt_rmsnorm_backward(dy, dys, h, hs, g, gd, rstd, dres, drs, rows, cols, dx, dg, ws, wb, None)

    _refused(bwd(cols=20), "multiple of 8")
    _refused(bwd(gd=3), "dtype")
    _refused(bwd(dg=None), "dgamma")
    _refused(bwd(dy=None), "null")
    _refused(bwd(rstd=None), "null")
    _refused(bwd(hs=32), "aligned rows")
    _refused(bwd(dres=p + 2, drs=64), "dres needs")
    _refused(bwd(dx=p + 2), "16-byte")
    _refused(bwd(ws=None), "workspace")
    _refused(bwd(wb=16), "too small")
    assert lib.mt_rmsnorm_backward_workspace(0, 64) == 0 and lib.mt_rmsnorm_backward_workspace(2, 64) == 2 * 64 * 4


def test_gated_entry_points_refuse(p):
    lib = _lib.load()

    def out(**kw):
        o = _lib.GatedOutputs()
        for k, v in kw.items():
            setattr(o, k, v)
        return ctypes.byref(o)

    def mx(x=p, sx=p, w=p, sw=p, up=None, M=2, F=128, K=64, act=0, o=out(h=p)):
        return lib.mt_gemm_gated_mxfp8(x, sx, w, sw, up, M, F, K, act, o, None)

    _refused(mx(K=48), "multiple of 32")
    _refused(mx(K=0), "multiple of 32")
    _refused(mx(F=72), "multiple of 32")
    _refused(mx(M=-1), "negative")
    _refused(mx(M=1 << 40), "out of range")
    _refused(mx(act=9), "activation")
    _refused(mx(o=None), "null outputs")
    _refused(mx(o=out()), "no output")
    _refused(mx(x=None), "null pointer")
    _refused(mx(F=96), "given apart")
    _refused(mx(w=p + 4), "16-byte")
    _refused(mx(o=out(h=p + 16)), "32-byte")
    _refused(mx(o=out(q=p)), "codes need s")
    _refused(mx(o=out(q=p, s=p, s_stride=3)), "codes need s")
    _refused(mx(o=out(h=p, s=p)), "without codes")
    assert mx(M=0, x=None) == 0 and mx(F=0, x=None) == 0
    rc = lib.mt_gemm_gated_nvfp4(p, p, None, p, p, None, p, 2, 128, 64, 0, out(h=p), None)
    _refused(rc, "abs-max")

    def gb(dh=p, ds=64, gu=p, rows=2, F=64, act=0, dgu=p, q=None, s=None, ss=4, qt=None, st=None, sts=1):
        return lib.mt_gated_backward(dh, ds, gu, rows, F, act, dgu, None, q, s, ss, None, qt, st, sts, None, None)

    _refused(gb(dgu=None), "no output")
    _refused(gb(q=p), "codes need s")
    _refused(gb(q=p, s=p, ss=3), "codes need s")
    _refused(gb(q=p, s=p, qt=p), "need s_t")
    _refused(gb(q=p, s=p, qt=p, st=p, sts=0), "need s_t")
    _refused(gb(q=p, s=p, st=p), "without transposed codes")
    _refused(gb(qt=p, st=p), "without codes")
    _refused(gb(q=p + 8, s=p), "16-byte")
    _refused(gb(rows=1 << 40), "out of range")

    _refused(gb(F=40), "multiple of 32")
    _refused(gb(act=5), "activation")
    _refused(gb(rows=-2), "negative")
    _refused(gb(dh=None), "null")
    _refused(gb(ds=32), "aligned rows")
    _refused(gb(gu=p + 8), "16-byte")
    assert gb(rows=0, dh=None) == 0


def test_front_end_refuses_cpu_tensors_and_unknown_activations():
    t = torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: kernels.rmsnorm(t, t[0]), lambda: kernels.rmsnorm_backward(t, t, t[0], t[:, 0]),
              lambda: kernels.gated_backward(t, t), lambda: kernels.gemm_gated_mxfp8(t, t, t, t),
              lambda: kernels.gemm_gated_nvfp4(t, t, t, t, t, t), lambda: RMSNorm(64, params_dtype=torch.bfloat16, device="cpu")(t),
              lambda: gated_linear(t, t, activation="relu", qlinear_params=MXFP8),
              lambda: GatedLinear(64, 64, activation="relu", device="cpu", qlinear_params=MXFP8),
              lambda: GatedLinear(64, 48, device="cpu", qlinear_params=MXFP8)):
        with pytest.raises(_lib.MtError):
            f()


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """With another device current, the wrapped call sees its tensors' device; errors restore the caller's."""
    current, seen = [0], []

    class FakeDevice:
        def __init__(self, d):
            self.d = d.index

        def __enter__(self):
            self.before, current[0] = current[0], self.d

        def __exit__(self, *a):
            current[0] = self.before

    class FakeTensor:
        is_cuda, device = True, torch.device("cuda", 1)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", FakeDevice)
    f = kernels._on_tensor_device(lambda t: seen.append(current[0]))
    f(FakeTensor())
    assert seen == [1] and current == [0]

    def boom(t):
        raise _lib.MtError("x")

    with pytest.raises(_lib.MtError):
        kernels._on_tensor_device(boom)(FakeTensor())
    assert current == [0]


def test_activation_values_match_the_header():
    import re
    text = open(_lib.HEADER_PATHS[0]).read()
    for name in ("MT_ACT_SILU", "MT_ACT_GELU"):
        assert int(re.search(name + r"\s*=\s*(\d+)", text).group(1)) == getattr(_lib, name)


def test_non_quantized_gated_linear_has_gradients():
    """The bf16 recipe runs on torch, on any device."""
    plain = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.NON_QUANTIZE)
    for act in ("silu", "gelu"):
        x, w = torch.randn(3, 32, dtype=torch.float64, requires_grad=True), torch.randn(64, 32, dtype=torch.float64, requires_grad=True)
        assert torch.autograd.gradcheck(lambda a, b: gated_linear(a, b, activation=act, qlinear_params=plain), (x, w))
