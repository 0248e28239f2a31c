"""float32 cross entropy on values whose products lose most of what the split into three bfloat16 leaves out, all in the same
direction: test_float32_split_cpu.py has the bound, one rounding of float32 a product, which the oracle's dz counts."""
import pytest
import torch

from test_decoder_gpu import F32, check, make

pytestmark = pytest.mark.gpu

WORST = 1 + 2.0 ** -8 - 2.0 ** -17


@pytest.mark.parametrize("rows", [7, 40, 130, 300])
@pytest.mark.parametrize("dim", [32, 384])
def test_products_that_lose_the_most(rows, dim):
    h, w, y = make(rows, dim, 391, F32, seed=rows, ignored=0.1)
    g = torch.Generator(device="cuda").manual_seed(dim)
    # powers of two times the same bits: losses of one sign where the signs of h and W agree, as they do in many rows of W
    size = torch.randint(-3, 1, h.shape, generator=g, device="cuda").float()
    h = WORST * 2.0 ** size * 0.25
    agree = (torch.rand(391, 1, generator=g, device="cuda") < 0.5).float()
    some = (torch.rand(391, dim, generator=g, device="cuda") < 0.5).float()
    w = WORST * 2.0 ** -5 * torch.where(agree > 0, 1.0, 1.0 - 2.0 * some)
    assert h.dtype == w.dtype == F32
    check(h, w, y, "none")
    check(h, w, y, "mean")
