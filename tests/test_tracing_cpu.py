"""Calls into the kernels' front end stay out of a compiler's graphs."""
import torch

from minitransformer_b200.module import config
from minitransformer_b200.module.gated_linear import GatedLinear, gated_linear
from test_norm_gated_cpu import _ExactOp

EXACT = config.QLinearParams(quantize=True, quantize_op=_ExactOp())


def _traced(f, *args):
    """Names of what a compiler would take over of f."""
    seen = []

    def backend(graph, _):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op.startswith("call"))
        return graph.forward

    torch._dynamo.reset()
    out = torch.compile(f, backend=backend)(*args)
    torch._dynamo.reset()
    return out, seen


def test_functional_and_modules_are_not_traced():
    x, w = torch.randn(32, 32).to(torch.bfloat16), torch.randn(64, 32).to(torch.bfloat16)
    lin = GatedLinear(32, 32, device="cpu", params_dtype=torch.bfloat16, qlinear_params=EXACT)
    for f in (lambda t: gated_linear(t + 1, w, qlinear_params=EXACT), lambda t: lin(t + 1)):
        with torch.no_grad():
            out, seen = _traced(f, x)
            assert torch.equal(out, f(x)) and len(seen) <= 1 and all("add" in s for s in seen), seen
