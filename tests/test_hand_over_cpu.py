"""What a layer hands on with its output (TensorCopies): its lifetime, and when the quantizer takes it."""
import copy
import gc
import pickle
import weakref

import pytest
import torch

from minitransformer_b200 import _lib, kernels
from minitransformer_b200.module import config
from minitransformer_b200.ops import quantization as Q
from minitransformer_b200.ops.mxfp8_quantize_op import Mxfp8QuantizeOp


def _copies(rows, cols, transposed=True):
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    return Q.QuantizeResult(u8(rows, cols), u8(rows, cols // 32), u8(cols, rows) if transposed else None,
                            u8(cols, rows // 32) if transposed else None)


def test_copies_live_as_long_as_their_tensor():
    y, made = torch.zeros(2, 16, 64, dtype=torch.bfloat16), _copies(32, 64)
    t = Q.TensorCopies(y, made)
    assert t.shape == (32, 64) and t.of(y.view(32, 64)) is made
    alive = weakref.ref(made.data)
    del made
    assert alive() is not None
    del y
    assert alive() is None and t.of(torch.zeros(32, 64, dtype=torch.bfloat16)) is None


def test_copies_leave_no_trace_on_their_tensor(tmp_path):
    y = torch.zeros(32, 64, dtype=torch.bfloat16)
    t = Q.TensorCopies(y, _copies(32, 64))
    torch.save(y, tmp_path / "y.pt")
    assert torch.equal(torch.load(tmp_path / "y.pt", weights_only=True), y) and t.of(y) is not None
    alive = weakref.ref(t.of(y).data)
    del t                                                    # the layer's next call
    assert alive() is None


def test_copies_of_a_tensor_that_only_autograd_holds():
    """The tensor's Python object goes and comes back while a graph holds it; the copies go with the graph."""
    w = torch.ones(32, 64, requires_grad=True)
    y = torch.zeros(32, 64)
    t = Q.TensorCopies(y, _copies(32, 64))
    alive = weakref.ref(t.of(y).data)
    out = (y * w).sum()                                      # saves y
    del y
    out.backward()
    del out
    gc.collect()
    assert alive() is None


def test_copies_count_for_their_tensor_unchanged():
    y, made = torch.zeros(32, 64, dtype=torch.bfloat16), _copies(32, 64)
    t = Q.TensorCopies(y, made)
    assert t.of(y.detach().reshape(32, 64)) is made and t.of(y.clone()) is None
    y[3].add_(1)
    assert t.of(y) is None
    with torch.inference_mode():
        z = torch.zeros(32, 64, dtype=torch.bfloat16)
        assert Q.TensorCopies(z, made).of(z) is made


def test_a_copied_or_pickled_holder_remembers_no_tensor():
    y = torch.zeros(32, 64, dtype=torch.bfloat16)
    t = Q.TensorCopies(y, _copies(32, 64))
    for u in (copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
        assert u.shape == (32, 64) and u.of(y) is None


def test_the_quantizer_takes_copies_only_where_they_hold(monkeypatch):
    calls = []

    def fake(x, return_transpose=True, into=None):
        calls.append(return_transpose)
        c = _copies(*x.shape, transposed=return_transpose)
        return kernels.Quantized(c.data, c.scale, c.scale, c.data_t, c.scale_t, c.scale_t)

    monkeypatch.setattr(kernels, "quantize_mxfp8", fake)
    op, p = Mxfp8QuantizeOp(), config.get_qlinear_params_from_predefined(config.QuantizeRecipe.MXFP8_SUB_CHANNEL).x_params
    y, made = torch.zeros(32, 64, dtype=torch.bfloat16), _copies(32, 64, transposed=False)
    meta = Q.QuantizeInputMeta(quantized=Q.TensorCopies(y, made))
    assert op.quantize(y, p, input_meta=meta) is made and not calls
    assert op.quantize(y.view(2, 16, 64), p, input_meta=meta) is made and not calls
    assert op.quantize(y, p, return_transpose=True, input_meta=meta).data_t is not None and calls == [True]
    op.quantize(y.clone(), p, input_meta=meta)                  # equal, but not that tensor: read again
    y.mul_(2)
    op.quantize(y, p, input_meta=meta)
    assert calls == [True, False, False]
    with pytest.raises(_lib.MtError, match="copies of"):
        op.quantize(y[:16], p, input_meta=meta)
    # a caller's own result counts as given
    own = _copies(32, 64)
    assert op.quantize(y, p, return_transpose=True, input_meta=Q.QuantizeInputMeta(quantized=own)) is own
    with pytest.raises(_lib.MtError, match="copies of"):
        op.quantize(y[:16], p, input_meta=Q.QuantizeInputMeta(quantized=own))
