"""The number of rows chooses the form of the 4-bit linear product: fewer rows may not take longer than more of them."""
import pytest
import torch

from test_gpu_padding_rows import milliseconds
from test_gpu_w4 import to, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [1024, 2048])
def test_linear_of_fewer_rows_takes_no_longer(dev, N, dtype):
    from mi355moe import w4
    g = torch.Generator().manual_seed(N)
    W = w4.W4Matrix(*to(dev, weights(g, N, 4096, 128, False)))
    x = torch.randn((300, 4096), generator=g).to(dtype).to(dev)
    few, many = (24, 90) if dtype == torch.float32 else (64, 300)
    t = [milliseconds(lambda: w4.linear(x[:m], W))[0] for m in (few, many)]
    assert t[0] <= 1.4 * t[1] + 0.002, f"{few} rows {t[0]} ms, {many} rows {t[1]} ms"
