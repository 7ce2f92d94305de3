"""CPU checks of the norm and gated entry points: refusals before anything reaches a GPU, and the device guard."""
import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from minitransformer_b200 import _lib, kernels
from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear, gated_linear
from minitransformer_b200.module.linear import Linear
from minitransformer_b200.module.rmsnorm import RMSNorm
from minitransformer_b200.ops import quantization as Q

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

    _refused(fwd(r=p, rs=72, h=p), "row stride to be cols")
    _refused(fwd(x=p, xs=128, r=p + 64, rs=64, h=p), "row stride to be cols")
    _refused(bwd(dres=p, drs=72), "row stride of cols")
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

    def gb(dh=p, ds=64, dr=2, gu=p, rows=2, F=64, act=0, dgu=p, q=None, s=None, ss=4, qt=None, st=None, sts=1):
        return lib.mt_gated_backward(dh, ds, dr, gu, rows, F, act, dgu, None, q, s, ss, None, qt, st, sts, None, None)

    _refused(gb(dgu=None), "no output")
    _refused(gb(dr=3), "rows for")
    _refused(gb(dr=0), "rows for")
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


def test_first_argument_may_be_named(monkeypatch):
    class FakeTensor:
        is_cuda, device = True, torch.device("cuda", 0)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    t = FakeTensor()
    f = kernels._on_tensor_device(lambda qa, other=1: (qa, other))
    assert f(qa=t, other=2) == (t, 2) and f(t) == (t, 1)
    with pytest.raises(_lib.MtError, match="qa is missing"):
        f(other=2)
    for g in (kernels.rmsnorm, kernels.rmsnorm_backward, kernels.gated_backward, kernels.gemm_gated_mxfp8, kernels.gemm_gated_nvfp4):
        with pytest.raises(_lib.MtError, match="is missing"):
            g()


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


class _ExactOp(Q.QuantizeOpBase):
    """Test double for the kernels: 'codes' are the values themselves in fp32, products are exact."""
    supports_allgather = False

    def quantize(self, x, qparams, return_transpose=False, reduce_amax=False, tp_group=None, input_meta=None):
        x = x.reshape(-1, x.shape[-1]).float().contiguous()
        one = torch.ones(1, 1)
        return Q.QuantizeResult(x, one, x.t().contiguous() if return_transpose else None, one if return_transpose else None)

    def qgemm(self, qx, qw, m_params, out_dtype, sx, sw, bias=None, out=None, accumulate=False, global_amax_qx=None,
              global_amax_qw=None, qparams_x=None, qparams_w=None):
        return (qx @ qw.t()).to(out_dtype)

    def gated_qgemm(self, qx, qw, sx, sw, activation, global_amax_qx=None, global_amax_qw=None, want_h=True, want_gu=False,
                    quantize_h=False, want_amax=False):
        gu = qx @ qw.t()
        g, u = gu.chunk(2, -1)
        return kernels.GatedResult((torch.nn.functional.silu(g) * u).to(torch.bfloat16), gu.to(torch.bfloat16) if want_gu else None)

    def gated_backward(self, dh, gu, qparams, activation):
        g, u = gu.float().chunk(2, -1)
        s = torch.sigmoid(g)
        dh = torch.nn.functional.pad(dh, (0, 0, 0, gu.shape[0] - dh.shape[0]))     # rows without a gradient
        dgu = torch.cat([dh.float() * u * s * (1 + g * (1 - s)), dh.float() * g * s], -1)
        return self.quantize(dgu, qparams, return_transpose=True)


def _column_parallel_worker(rank, world, port, result):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.manual_seed(0)
        bf = torch.bfloat16
        T, H, F = 40, 32, 128                          # 40 tokens: continued with zeros to 64
        x, dy = torch.randn(T, H).to(bf), torch.randn(T, H).to(bf)
        wg, wu, w2 = (torch.randn(*s).mul(0.2).to(bf) for s in ((F, H), (F, H), (H, F)))
        p = config.QLinearParams(quantize=True, quantize_op=_ExactOp())
        kw = dict(params_dtype=bf, device="cpu", qlinear_params=p, tp_group=dist.group.WORLD)
        fc1 = GatedLinear(H, F, parallel_mode="column", **kw)
        fc2 = Linear(F, H, parallel_mode="row", bias=False, **kw)
        assert fc1.weight.shape == (2 * F // world, H) and fc1.weight.tensor_model_parallel and fc1.weight.partition_dim == 0
        with torch.no_grad():
            fc1.weight.copy_(torch.cat([wg.chunk(world, 0)[rank], wu.chunk(world, 0)[rank]]))
            fc2.weight.copy_(w2.chunk(world, 1)[rank])
        xs = x.clone().requires_grad_()
        y = fc2(fc1(xs))
        y.backward(dy)
        X, G, U, W = (t.double().requires_grad_() for t in (x, wg, wu, w2))
        ref = (torch.nn.functional.silu(X @ G.t()) * (X @ U.t())) @ W.t()
        ref.backward(dy.double())
        rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
        tol = 4 * 2.0 ** -8      # at most four roundings to bf16 on the way to any of these
        grad1 = torch.cat([G.grad.chunk(world, 0)[rank], U.grad.chunk(world, 0)[rank]])
        errs = [rel(y, ref), rel(xs.grad, X.grad), rel(fc1.weight.grad, grad1), rel(fc2.weight.grad, W.grad.chunk(world, 1)[rank])]
        result[rank] = errs if max(errs) > tol else True
    finally:
        dist.destroy_process_group()


def test_column_parallel_gated_linear_on_two_ranks():
    """Each rank holds [gate shard; up shard]; dgrad is summed over the ranks."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    with mp.get_context("spawn").Manager() as m:
        result = m.dict()
        mp.spawn(_column_parallel_worker, args=(2, port, result), nprocs=2, join=True)
        assert dict(result) == {0: True, 1: True}, dict(result)


def test_mx_scale_rule_on_every_bf16_magnitude():
    """The scale rule of the register quantizer (integer arithmetic on bf16 bits), restated, against its definition."""
    import math
    from fractions import Fraction
    import numpy as np
    for bits in range(0x7F80):
        E = max((bits + 0x1F) >> 7, 8)
        value = Fraction(float(np.array([bits << 16], dtype=np.uint32).view(np.float32)[0]))
        e = -127
        if value:
            e = math.ceil(math.log2(value / 448)) - 2
            while Fraction(2) ** e < value / 448:
                e += 1
            e = max(e, -127)
        assert E - 8 == e + 127, hex(bits)
