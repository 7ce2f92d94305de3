"""More refusals of the norm and the gated entry points, before anything reaches a GPU."""
import pytest
import torch

from minitransformer_b200 import _lib, kernels


def test_gated_projection_refuses_options_of_the_plain_gemm():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    scales = [u8(kernels.swizzled_scale_bytes(r, 2)) for r in (4, 256)]

    def call():
        return kernels._gemm_gated("mxfp8", u8(4, 64), scales[0], None, u8(256, 64), scales[1], None, "silu", None, True, False, False, False)

    for options in (dict(d_amax=torch.zeros(1)), dict(scatter=([0, 0], 0, 2))):
        with kernels.gemm_options(**options):
            with pytest.raises(_lib.MtError, match="plain GEMMs"):
                call()
