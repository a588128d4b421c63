"""Refusals of the extension on the GPU: an argument check that fails raises, also where its message holds numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gemm_refuses_mismatched_shapes():
    from trenowanie_generatora_obrazkow_b200.ops._ext import err_buf, ext
    a = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    b = torch.zeros(64, 128, device="cuda", dtype=torch.bfloat16)
    c = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gemm"):
        ext().gemm(a, b, c, False, False, None, 1.0, 0.0, False, err_buf("cuda"))
