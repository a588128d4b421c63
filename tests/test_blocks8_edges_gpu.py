"""8-bit block operators at their edges on the GPU: scales far out."""
import pytest
import torch
from test_blocks8_gpu import held

from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
from trenowanie_generatora_obrazkow_b200.ops._ext import check_errors

pytestmark = pytest.mark.gpu
DEV = "cuda"
WIDE = [torch.bfloat16, torch.float32]  # types with fp32's range


@pytest.fixture(autouse=True)
def _no_kernel_errors():
    yield
    if torch.cuda.is_available():
        check_errors(DEV)


# ---------------------------------------------------------------------------------------------------------- far scales
@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 130])
def test_scales_whose_product_is_out_of_range(M, dtype):
    """The largest values of x's and W's blocks do not meet: the scales' product is beyond fp32, the sums are not."""
    x, w = torch.zeros(M, 256, device=DEV), torch.zeros(5, 256, device=DEV)
    x[:, 0], x[:, 1], x[:, 130] = 2.0 ** 100, 2.0 ** 84, 1.0
    w[:, 2] = 2.0 ** 60                   # beside x's zeros
    w[1, 1] = 2.0 ** 43                   # 2^127
    w[2, 1], w[2, 130] = -(2.0 ** 43), 3.0  # -2^127
    w[3, 130] = 5.0                       # 5, from the second block alone
    got = B8.linear_blocks(x.to(dtype), B8.quantize_blocks(w))
    want = (held(x) @ held(w).t()).to(dtype)
    assert want[0].tolist() == [0.0, 2.0 ** 127, -(2.0 ** 127), 5.0, 0.0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 130])
@pytest.mark.parametrize("e", [-149, -150, -154])
def test_scales_whose_product_is_too_small(M, dtype, e):
    """Sums of 49 2^19 2^e, normal numbers of fp32, from scales whose product is not."""
    x = torch.full((M, 128), 448 * 2.0 ** -70, device=DEV, dtype=dtype)
    w = torch.full((3, 128), 448 * 2.0 ** (e + 70), device=DEV)
    x[:, 64:], w[1, :64] = 0, 0
    got = B8.linear_blocks(x, B8.quantize_blocks(w))
    want = torch.tensor([49 * 2.0 ** (18 + e), 0.0, 49 * 2.0 ** (18 + e)], device=DEV, dtype=torch.float64).to(dtype)
    assert torch.equal(got, want.expand(M, 3))
