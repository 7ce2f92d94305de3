"""The operators of the pre-norm gated feed-forward block, as cases to be measured.

Three operators that a transformer block runs around its quantized linear layers:

  norm / norm_grad    residual addition, root-mean-square norm and its MXFP8 copies; the norm's gradients
  gate / gate_step    both projections of a gated feed-forward block with the activation and the product,
                      on MXFP8 or NVFP4 operands; the same with its whole backward pass
  gate_grad           gradient of activation and product, quantized to MXFP8 both ways

`run` computes them in elementary torch operations (own = False) or by the calls that a user of
minitransformer_b200 makes (own = True).
"""
import math

import torch

own = False

EPS = 1e-5
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decode step: residual stream in, row-wise codes for the next projection out
        dict(name="norm_token", op="norm", rows=1, cols=4096, residual=True, y=False, transpose=False),
        # a training step's norm at the decoder's width: bf16 output and both copies
        dict(name="norm_train", op="norm", rows=8192, cols=4096, residual=True, y=True, transpose=True),
        # a short odd batch: no gradient comes in along the residual stream
        dict(name="norm_grad_ragged", op="norm_grad", rows=1021, cols=2080, residual=False),
        # a training step's norm gradient at the tensor-parallel MLP's width
        dict(name="norm_grad_train", op="norm_grad", rows=8192, cols=8192, residual=True),
        # decode: the weights are read once for one token; the result feeds the next projection in 8 bits
        dict(name="gate_token", op="gate", fmt="mxfp8", rows=1, cols=4096, ffn=14336, act="silu", out="mxfp8"),
        # a decode batch
        dict(name="gate_batch", op="gate", fmt="mxfp8", rows=64, cols=4096, ffn=14336, act="silu", out="mxfp8"),
        # a ragged prompt through a small expert-sized block, gelu
        dict(name="gate_prompt", op="gate", fmt="mxfp8", rows=1000, cols=2048, ffn=768, act="gelu", out="bf16"),
        # a training forward pass on 4-bit operands: output and saved projections
        dict(name="gate_fp4_train", op="gate", fmt="nvfp4", rows=8192, cols=4096, ffn=14336, act="silu", out="train"),
        # gradient of activation and product, odd row count and a feature count that no tile divides
        dict(name="gate_grad_ragged", op="gate_grad", rows=1021, ffn=1376, act="gelu"),
        # the same at a training step's size
        dict(name="gate_grad_train", op="gate_grad", rows=8192, ffn=14336, act="silu"),
        # whole training pass of a small layer: forward, gradients of input and weight
        dict(name="gate_step_small", op="gate_step", rows=512, cols=1024, ffn=768, act="gelu"),
        # whole training pass at the decoder's size
        dict(name="gate_step", op="gate_step", rows=8192, cols=4096, ffn=14336, act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _by32(rng, lo, hi):
    return max(lo, _log(rng, lo, hi) // 32 * 32)


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "gate", "gate", "gate_grad", "gate_step"])
    act = rng.choice(["silu", "gelu"])
    if op == "norm":
        cols = _by32(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, min(16384, (1 << 26) // cols)), cols=cols, residual=rng.random() < 0.7,
                    y=rng.random() < 0.5, transpose=rng.random() < 0.5)
    if op == "norm_grad":
        cols = _by32(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, min(16384, (1 << 26) // cols)), cols=cols, residual=rng.random() < 0.7)
    if op == "gate_grad":
        ffn = _by32(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, min(16384, (1 << 26) // ffn)), ffn=ffn, act=act)
    cols, ffn = _by32(rng, 128, 8192), _by32(rng, 128, 16384)
    most = min(8192, (1 << 37) // (cols * ffn))
    if op == "gate":
        return dict(op=op, fmt=rng.choice(["mxfp8", "mxfp8", "nvfp4"]), rows=_log(rng, 1, most), cols=cols, ffn=ffn,
                    act=act, out=rng.choice(["mxfp8", "bf16", "train"]))
    return dict(op=op, rows=_log(rng, 16, most), cols=cols, ffn=ffn, act=act)


# ---------------------------------------------------------------------------------------------
# block formats, in elementary operations (float32 or float64 throughout)
# ---------------------------------------------------------------------------------------------
def _exponent_bits(e, like):
    """2^e for integer e in [-126, 127], exactly."""
    if like.dtype == torch.float64:
        return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _mx_rows(t):
    """t [R, C] (values of bf16) -> E4M3 codes [R, C] and E8M0 bytes [R, ceil(C / 32)] of 1x32 blocks."""
    rows, cols = t.shape
    blocks = (cols + 31) // 32
    v = torch.nn.functional.pad(t, (0, blocks * 32 - cols)).view(rows, blocks, 32)
    m, e = torch.frexp(v.abs().amax(-1))                    # 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).to(e.dtype)                     # ceil(log2(amax / 448))
    e = torch.where(m == 0, torch.full_like(e, -127), e).clamp(-127, 126)
    v = (v * _exponent_bits(-e, v)[..., None]).clamp(-448, 448)
    codes = v.to(torch.float32).to(torch.float8_e4m3fn).view(rows, blocks * 32)[:, :cols]
    return codes.contiguous(), (e + 127).to(torch.uint8)


def _gemm_layout(s):
    """Scale bytes [R, B] -> the order in which the block-scaled GEMM reads them: chunks of 128 rows x 4 blocks, byte
    (r % 32) * 16 + (r / 32) * 4 + b % 4, zero padded, chunk count along B a multiple of 4."""
    rows, blocks = s.shape
    rb, kc = (rows + 127) // 128, ((blocks + 3) // 4 + 3) // 4 * 4
    s = torch.nn.functional.pad(s, (0, kc * 4 - blocks, 0, rb * 128 - rows))
    return s.view(rb, 4, 32, kc, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _mx_copies(t, transpose):
    """What a user receives as the MXFP8 form of t: codes and scales, row-wise and (optionally) transposed."""
    q, s = _mx_rows(t)
    out = {"q": q, "s": s, "s_gemm": _gemm_layout(s)}
    if transpose:
        qt, st = _mx_rows(t.t().contiguous())
        out.update(qt=qt, st=st, st_gemm=_gemm_layout(st))
    return out


def _mx_values(q, s, dtype):
    """Codes and scale bytes -> the values they stand for."""
    rows, cols = q.shape
    blocks = s.shape[1]
    v = torch.nn.functional.pad(q.to(torch.float32).to(dtype), (0, blocks * 32 - cols)).view(rows, blocks, 32)
    f = _exponent_bits((s.to(torch.int32) - 127).clamp(min=-126), v)
    return (v * f[..., None]).view(rows, blocks * 32)[:, :cols]


def _as_values(copies):
    """8-bit tensors under the types whose values they hold."""
    return {k: (v.view(torch.float8_e8m0fnu) if k.startswith("s") else v) for k, v in copies.items()}


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nv_rows(t):
    """t [R, C] -> packed E2M1 codes [R, C / 2] (even column in the low nibble), E4M3 scale bytes [R, C / 16], max |t|."""
    rows, cols = t.shape
    amax = t.abs().amax().reshape(1).float()
    v = t.view(rows, cols // 16, 16)
    s = (v.abs().amax(-1) / 6 * (2688.0 / amax)).clamp(max=448).to(torch.float8_e4m3fn)
    scaled = v * (2688.0 / amax / s.float().clamp(min=1e-30))[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=t.device)
    code = torch.bucketize(scaled.abs().clamp(max=6), edges) + 8 * (scaled < 0)
    code = code.view(rows, cols).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), s.view(torch.uint8), amax


def _nv_values(q, s, amax, dtype):
    rows = q.shape[0]
    table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=dtype, device=q.device)
    v = torch.stack([table[(q & 15).long()], table[(q >> 4).long()]], dim=-1).view(rows, -1, 16)
    return (v * s.view(torch.float8_e4m3fn).to(torch.float32).to(dtype)[..., None]).view(rows, -1) * (amax.to(dtype) / 2688.0)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _randn(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c = dict(case)
    op, rows = c["op"], c["rows"]
    if op in ("norm", "norm_grad"):
        # a residual stream has a few channels far above the rest
        scale = 0.5 + 4.0 * (torch.rand(c["cols"], generator=gen, device="cuda") < 0.01)
        c["x"] = (torch.randn(rows, c["cols"], generator=gen, device="cuda") * scale).to(torch.bfloat16)
        c["gamma"] = (1 + 0.2 * torch.randn(c["cols"], generator=gen, device="cuda")).to(torch.bfloat16)
        if op == "norm":
            c["r"] = _randn(gen, rows, c["cols"]) if c["residual"] else None
        else:
            c["rstd"] = torch.rsqrt(c["x"].float().square().mean(-1) + EPS)
            c["dy"] = _randn(gen, rows, c["cols"], std=1e-3)
            c["dh"] = _randn(gen, rows, c["cols"], std=1e-3) if c["residual"] else None
    elif op == "gate":
        # quantized activations (the norm's output) and the quantized [gate; up] weight that a server or a
        # training step holds
        x, w = _randn(gen, rows, c["cols"]), _randn(gen, 2 * c["ffn"], c["cols"], std=0.02)
        for k, t in (("x", x), ("w", w)):
            if c["fmt"] == "mxfp8":
                c["q" + k], c["s" + k] = _mx_rows(t.float())
                c["q" + k] = c["q" + k].view(torch.uint8)
            else:
                c["q" + k], c["s" + k], c["amax" + k] = _nv_rows(t.float())
            c["sg" + k] = _gemm_layout(c["s" + k])
    elif op == "gate_grad":
        c["gu"] = _randn(gen, rows, 2 * c["ffn"], std=1.3)
        c["dh"] = _randn(gen, rows, c["ffn"], std=1e-3)
    else:
        c["x"] = _randn(gen, rows, c["cols"])
        c["w"] = _randn(gen, 2 * c["ffn"], c["cols"], std=0.02)
        c["dh"] = _randn(gen, rows, c["ffn"], std=1e-3)
    return c


# ---------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------
def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    t = torch.tanh(GELU_C * (g + GELU_A * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * GELU_C * (1 + 3 * GELU_A * g * g)


def _bf16(t):
    return t.to(torch.bfloat16)


def _plain_norm(c):
    h = c["x"] if c["r"] is None else _bf16(c["x"].float() + c["r"].float())
    v = h.float()
    rstd = 1 / torch.sqrt((v * v).mean(-1) + EPS)
    y = _bf16(v * rstd[:, None] * c["gamma"].float())
    out = {"rstd": rstd, **_as_values(_mx_copies(y.float(), c["transpose"]))}
    if c["r"] is not None:
        out["h"] = h
    if c["y"]:
        out["y"] = y
    return out


def _plain_norm_grad(c):
    v, rstd, dy = c["x"].float(), c["rstd"][:, None], c["dy"].float()
    xhat, a = v * rstd, dy * c["gamma"].float()
    dx = rstd * (a - xhat * (a * xhat).mean(-1, keepdim=True))
    if c["dh"] is not None:
        dx = dx + c["dh"].float()
    return {"dx": _bf16(dx), "dgamma": (dy * xhat).sum(0)}


def _gate_out(gu, c):
    f = c["ffn"]
    h = _bf16(_act(gu[:, :f], c["act"])[0] * gu[:, f:])
    if c["out"] == "mxfp8":
        return _as_values(_mx_copies(h.float(), False))
    if c["out"] == "bf16":
        return {"h": h}
    return {"h": h, "gu": _bf16(gu)}


def _plain_gate(c):
    if c["fmt"] == "mxfp8":
        x, w = (_mx_values(c["q" + k].view(torch.float8_e4m3fn), c["s" + k], torch.float32) for k in "xw")
    else:
        x, w = (_nv_values(c["q" + k], c["s" + k], c["amax" + k], torch.float32) for k in "xw")
    return _gate_out(x @ w.t(), c)


def _gate_gradient(gu, dh, act):
    """[dg | du] in bf16 from the saved projections."""
    f = dh.shape[1]
    a, d = _act(gu[:, :f], act)
    return _bf16(torch.cat([dh * gu[:, f:] * d, dh * a], dim=1))


def _plain_gate_grad(c):
    return _as_values(_mx_copies(_gate_gradient(c["gu"].float(), c["dh"].float(), c["act"]).float(), True))


def _plain_gate_step(c):
    f = c["ffn"]
    values = lambda t: _mx_values(*_mx_rows(t.float()), torch.float32)  # noqa: E731
    x, w = values(c["x"]), values(c["w"])
    xt, wt = values(c["x"].t().contiguous()), values(c["w"].t().contiguous())
    gu = x @ w.t()
    h = _bf16(_act(gu[:, :f], c["act"])[0] * gu[:, f:])
    dgu = _gate_gradient(_bf16(gu).float(), c["dh"].float(), c["act"])      # projections are saved in bf16
    return {"h": h, "dx": _bf16(values(dgu) @ wt.t()), "dw": _bf16(values(dgu.t().contiguous()) @ xt.t())}


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------
def _own_copies(q, transpose=False):
    out = {"q": q.data.view(torch.float8_e4m3fn), "s": q.scale, "s_gemm": q.scale_swz}
    if transpose:
        out.update(qt=q.data_t.view(torch.float8_e4m3fn), st=q.scale_t, st_gemm=q.scale_t_swz)
    return _as_values(out)


def _own_run(c):
    from minitransformer_b200 import kernels
    op = c["op"]
    if op == "norm":
        r = kernels.rmsnorm(c["x"], c["gamma"], EPS, residual=c["r"], want_y=c["y"], return_transpose=c["transpose"])
        out = {"rstd": r.rstd, **_own_copies(r.quantized, c["transpose"])}
        if c["r"] is not None:
            out["h"] = r.h
        if c["y"]:
            out["y"] = r.y
        return out
    if op == "norm_grad":
        dx, dgamma = kernels.rmsnorm_backward(c["dy"], c["x"], c["gamma"], c["rstd"], dresidual=c["dh"])
        return {"dx": dx, "dgamma": dgamma}
    if op == "gate":
        want = dict(activation=c["act"], want_h=c["out"] != "mxfp8", want_gu=c["out"] == "train",
                    quantize_h=c["out"] == "mxfp8")
        if c["fmt"] == "mxfp8":
            r = kernels.gemm_gated_mxfp8(c["qx"], c["sgx"], c["qw"], c["sgw"], sb_lin=c["sw"], **want)
        else:
            r = kernels.gemm_gated_nvfp4(c["qx"], c["sgx"], c["amaxx"], c["qw"], c["sgw"], c["amaxw"], sb_lin=c["sw"], **want)
        if c["out"] == "mxfp8":
            return _own_copies(r.quantized)
        return {"h": r.h} if c["out"] == "bf16" else {"h": r.h, "gu": r.gu}
    if op == "gate_grad":
        return _own_copies(kernels.gated_backward(c["dh"], c["gu"], activation=c["act"]).quantized, True)
    from minitransformer_b200.module import config
    from minitransformer_b200.module.gated_linear import gated_linear
    params = config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL)
    x, w = c["x"].detach().requires_grad_(), c["w"].detach().requires_grad_()
    h = gated_linear(x, w, activation=c["act"], qlinear_params=params)
    dx, dw = torch.autograd.grad(h, (x, w), c["dh"])
    return {"h": h, "dx": dx, "dw": dw}


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "gate": _plain_gate, "gate_grad": _plain_gate_grad,
          "gate_step": _plain_gate_step}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    m = case["rows"]
    op = case["op"]
    if op == "norm":
        n = m * case["cols"]
        by = 2 + (4 if case["residual"] else 0) + (2 if case["y"] else 0) + (1 + 2 / 32) * (2 if case["transpose"] else 1)
        return {"bytes": n * by + 4 * m + 2 * case["cols"], "flops": 8 * n}
    if op == "norm_grad":
        n = m * case["cols"]
        return {"bytes": n * (8 if case["residual"] else 6) + 4 * m + 6 * case["cols"], "flops": 12 * n}
    f = case["ffn"]
    if op == "gate_grad":
        return {"bytes": m * f * (6 + 4 * (1 + 2 / 32)), "flops": 30 * m * f}
    k = case["cols"]
    if op == "gate":
        per = 1 + 1 / 32 if case["fmt"] == "mxfp8" else 0.5 + 1 / 16
        out = {"mxfp8": 1 + 2 / 32, "bf16": 2, "train": 6}[case["out"]]
        return {"bytes": (m + 2 * f) * k * per + m * f * out, "flops": 4.0 * m * f * k}
    # x, w and dh in, h, dx and dw out; the projections are saved and read once
    return {"bytes": 2 * (2 * m * k + 4 * f * k + 2 * m * f) + 8 * m * f, "flops": 12.0 * m * f * k}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_blocks(t):
    """Values of bf16 in float64, [R, C] -> (E4M3 code values, 2^e) of 1x32 blocks: e is the smallest integer with
    amax <= 448 * 2^e, the code the nearest E4M3 value of t / 2^e, ties to the even mantissa."""
    rows, cols = t.shape
    t = torch.cat([t, t.new_zeros(rows, -cols % 32)], 1)
    power = torch.tensor([2.0 ** k for k in range(-127, 128)], dtype=torch.float64, device=t.device)
    amax = t.abs().reshape(rows, -1, 32).max(-1).values
    scale = power[torch.bucketize(amax, 448 * power).clamp(max=254)]          # first power with amax <= 448 * power
    v = t / scale.repeat_interleave(32, 1)
    # spacing of E4M3 around v: 2^(floor(log2 |v|) - 3), 2^-9 below 2^-6; torch.round takes ties to even
    step = power[torch.bucketize(v.abs(), power, right=True).clamp(min=122) - 1] / 8
    return (torch.round(v / step) * step)[:, :cols], scale


def _exact_values(t):
    q, s = _exact_blocks(t)
    return q * s.repeat_interleave(32, 1)[:, :q.shape[1]]


def _exact_copies(t, transpose):
    out = {}
    for tag, v in (("", t),) + ((("t", t.t()),) if transpose else ()):
        q, s = _exact_blocks(v)
        # padding of the GEMM layout holds byte 0, which stands for 2^-127
        rows, blocks = s.shape
        full = torch.full(((rows + 127) // 128 * 128, (blocks + 15) // 16 * 16), 2.0 ** -127, dtype=torch.float64, device=s.device)
        full[:rows, :blocks] = s
        lay = full.reshape(full.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).reshape(-1)
        out.update({"q" + tag: q, "s" + tag: s, "s" + tag + "_gemm": lay})
    return out


def _exact_act(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    inner = GELU_C * (g + GELU_A * g ** 3)
    cosh = torch.cosh(inner.clamp(-300, 300))
    return g * torch.sigmoid(2 * inner), torch.sigmoid(2 * inner) + 0.5 * g * GELU_C * (1 + 3 * GELU_A * g ** 2) / cosh ** 2


def _r16(t):
    return t.to(torch.bfloat16).double()


def exact(case, seed):
    c = prepare(case, seed)
    op = c["op"]
    if op == "norm":
        h = c["x"].double() if c["r"] is None else _r16(c["x"].double() + c["r"].double())
        rstd = ((h ** 2).sum(1) / h.shape[1] + EPS) ** -0.5
        y = h * rstd.unsqueeze(1) * c["gamma"].double()
        out = {"rstd": rstd, **_exact_copies(_r16(y), c["transpose"])}
        if c["r"] is not None:
            out["h"] = c["x"].double() + c["r"].double()
        if c["y"]:
            out["y"] = y
        return out
    if op == "norm_grad":
        h, dy, r = c["x"].double(), c["dy"].double(), c["rstd"].double().unsqueeze(1)
        gdy = c["gamma"].double() * dy
        dx = r * gdy - r ** 3 * h * (gdy * h).sum(1, keepdim=True) / h.shape[1]
        if c["dh"] is not None:
            dx += c["dh"].double()
        return {"dx": dx, "dgamma": torch.einsum("mk,mk,m->k", dy, h, r[:, 0])}
    if op == "gate_grad":
        g, u = c["gu"].double().split(c["ffn"], 1)
        a, d = _exact_act(g, c["act"])
        dgu = torch.cat([c["dh"].double() * u * d, c["dh"].double() * a], 1)
        return _exact_copies(_r16(dgu), True)
    f = c["ffn"]
    if op == "gate":
        if c["fmt"] == "mxfp8":
            x, w = (c["q" + k].view(torch.float8_e4m3fn).float().double()
                    * (2.0 ** (c["s" + k].double() - 127)).repeat_interleave(32, 1) for k in "xw")
        else:
            grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
            sides = []
            for k in "xw":
                n = torch.stack([c["q" + k] & 15, c["q" + k] >> 4], 2).flatten(1).long()
                v = grid[n % 8] * (1 - 2 * (n // 8)).double()
                s = c["s" + k].view(torch.float8_e4m3fn).float().double().repeat_interleave(16, 1)
                sides.append(v * s * c["amax" + k].double() / (6 * 448))
            x, w = sides
        g, u = x @ w[:f].t(), x @ w[f:].t()
        h = _exact_act(g, c["act"])[0] * u
        if c["out"] == "mxfp8":
            return _exact_copies(_r16(h), False)
        if c["out"] == "bf16":
            return {"h": h}
        return {"h": h, "gu": torch.cat([g, u], 1)}
    x, w, dh = c["x"].double(), c["w"].double(), c["dh"].double()
    wq = _exact_values(w)
    g, u = (_exact_values(x) @ wq.t()).split(f, 1)
    h = _exact_act(g, c["act"])[0] * u
    g, u = _r16(g), _r16(u)                                   # what the backward pass is given
    a, d = _exact_act(g, c["act"])
    dgu = _r16(torch.cat([dh * u * d, dh * a], 1))
    del wq
    return {"h": h, "dx": _exact_values(dgu) @ _exact_values(w.t()).t(),
            "dw": _exact_values(dgu.t()) @ _exact_values(x.t()).t()}
