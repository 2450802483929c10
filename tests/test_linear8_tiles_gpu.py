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


# G by LDS-DMA where N is a multiple of 8 (bfloat16), through registers otherwise: 256-wide tiles over one to six stages with a ragged last one, and sides
# narrower than half a tile
WGRADS = [(200, 3592, 3329), (333, 3504, 3600), (64, 3504, 3600), (130, 3590, 3400), (300, 24, 25100), (300, 50000, 24), (2352, 200, 50000)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["dense", "slab"])
@pytest.mark.parametrize("M,N,K", WGRADS)
def test_wgrad_of_large_and_narrow_operands(device, M, N, K, layout, dtype):
    from speedplusbaseline_amd import ops
    G, X8 = data(M, N, dtype, M, layout, scale=1e-3), ops.quant8(data(M, K, torch.bfloat16, N))
    first = ops.gemm8_wgrad(G, X8)
    check_wgrad(G, X8, first)
    assert torch.equal(first, ops.gemm8_wgrad(G, X8))
    wide = torch.randn(N, K + 5, device="cuda")
    before = wide.clone()
    out = ops.gemm8_wgrad(G, X8, dW=wide[:, 2:2 + K])
    check_wgrad(G, X8, out, before[:, 2:2 + K].double())
    assert torch.equal(wide[:, :2], before[:, :2]) and torch.equal(wide[:, 2 + K:], before[:, 2 + K:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_wgrad_rows_and_columns_behind_the_matrix_do_not_count(device, dtype):
    """ragged ends in a matrix of NaN: rows behind the last one, columns beside G"""
    from speedplusbaseline_amd import ops
    M, N, K = 200, 3592, 3400
    wide = torch.full((M + 60, N + 8), float("nan"), dtype=dtype, device="cuda")
    wide[:M, :N] = data(M, N, dtype, 3, scale=1e-3)
    X8 = ops.quant8(data(M, K, torch.bfloat16, 4))
    dw = ops.gemm8_wgrad(wide[:M, :N], X8)
    assert dw.isfinite().all() and torch.equal(dw, ops.gemm8_wgrad(wide[:M, :N].contiguous(), X8))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,N,K", [(3, 8, 130), (70, 40, 300), (2400, 1024, 1200), (70, 3504, 3600), (70, 3501, 3600)])
def test_wgrad_of_infinite_gradients(device, M, N, K, dtype):
    """infinities of the same places and signs as in the sum of products itself, whatever the type; NaN where they meet a zero or each other"""
    from speedplusbaseline_amd import ops
    G, x = data(M, N, dtype, M, scale=1e-3), data(M, K, torch.bfloat16, N)
    G[1, 2], G[2, 5], G[0, 5], G[2, 7] = float("inf"), -float("inf"), float("inf"), float("nan")
    X8 = ops.quant8(x)
    dw = ops.gemm8_wgrad(G, X8)
    want = G.double().t() @ ops.dequant8(X8, torch.float32).double()
    assert want[2].isinf().any() and want[5].isnan().any() and want[7].isnan().all()
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(dw), f(want)), f.__name__


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (16, 513, 1001), (5, 40, 17000), (2, 16, 64)])
def test_few_rows_have_exact_products(device, M, N, K, dtype):
    """a 16-bit result of up to 16 rows is the float32 one rounded once"""
    from speedplusbaseline_amd import ops
    A, (B, _) = ops.quant8(data(M, K, torch.bfloat16, M, scale=0.02)), ops.quant8_weight(data(N, K, torch.float32, N, scale=0.02), transpose=False)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(2)).cuda()
    y = ops.gemm8(A, B, bias=bias, dtype=torch.float32)
    check_product(A, B, bias, y)
    assert torch.equal(ops.gemm8(A, B, bias=bias, dtype=dtype), y.to(dtype))
