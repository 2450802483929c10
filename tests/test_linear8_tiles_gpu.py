"""The forms of the 8-bit products that only large or narrow operands reach, each several stages deep with ragged ends, against float64 (bounds: test_linear8_gpu.py)."""
import pytest
import torch

from test_linear8_gpu import TYPES, check_product, check_wgrad, data

pytestmark = pytest.mark.gpu

# two tiles of 128 on a compute unit, nine steps; 256-wide tiles, twelve steps; sides that fill a fifth of a tile
LARGE = [(3700, 1300, 1100), (3329, 3841, 1500), (40000, 24, 144), (40000, 24, 1300), (24, 40000, 700), (19000, 200, 600), (70, 20000, 1100)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K", LARGE)
def test_product_of_large_and_narrow_operands(device, M, N, K, dtype):
    from speedplusbaseline_amd import ops
    A, (B, _) = ops.quant8(data(M, K, torch.bfloat16, M, scale=0.02)), ops.quant8_weight(data(N, K, torch.float32, N, scale=0.02), transpose=False)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(2)).cuda()
    y = ops.gemm8(A, B, bias=bias, dtype=dtype)
    check_product(A, B, bias, y)
    wide = torch.full((M, N + 9), 7.0, dtype=dtype, device="cuda")
    assert torch.equal(ops.gemm8(A, B, bias=bias, dtype=dtype, Y=wide[:, 5:5 + N]), y) and (wide[:, :5] == 7).all() and (wide[:, 5 + N:] == 7).all()
