"""Layer norm backward over many rows: the order of the sums over rows.  U = 2^-24, the rounding of a float32 addition."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("M,C", [(200000, 8200), (70001, 8193), (1000, 20000)])
def test_sums_over_many_long_rows(device, M, C, dtype):
    """One row of x and of g for all M (stride 0), so that every column adds M equal terms, which round in one direction as long as the sum stays in a binade.
    At most 64 ranges of rows, in each of them blocks of 64, then the ranges: 64 + M / 4096 + 1 + 4 + 16 additions deep; a term of dgamma carries
    three roundings of its own, and mean and rstd are inputs."""
    from speedplusbaseline_amd import ops
    gen = torch.Generator().manual_seed(M)
    x = torch.randn(1, C, generator=gen).to(dtype).cuda()
    g = (1 + torch.rand(1, C, generator=gen)).to(dtype).cuda()
    _, mean, rstd = ops.layernorm_fwd(x)
    m, r = mean.expand(M).contiguous(), rstd.expand(M).contiguous()
    dx, dgamma, dbeta = ops.layernorm_bwd(g.expand(M, C), x.expand(M, C), m, r)
    one = ops.layernorm_bwd(g, x, mean, rstd)[0]
    assert (dx[:100] == one).all() and (dx[-100:] == one).all()
    depth = 64 + M / 4096 + 1 + 4 + 16
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    want_g, want_b = (M * g.double() * xh)[0], (M * g.double())[0]
    off_x = U * (x.double().abs() + mean.double().abs()) * rstd.double()[:, None]              # of x - mean
    assert ((dbeta.double() - want_b).abs() <= depth * U * want_b.abs()).all()
    assert ((dgamma.double() - want_g).abs() <= (depth + 3) * U * want_g.abs() + (M * g.double() * off_x)[0]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("M,C", [(8000, 64), (2000, 1001), (500, 4096), (1, 24)])
def test_partial_sums_are_joined_without_further_roundings(device, M, C, dtype):
    """At most 512 workgroups' worth of rows, all of them the same one: a thread has one term, so of dbeta only the partial rows and the result are rounded,
    a rounding each (U * sum of the partial rows + U * result)."""
    from speedplusbaseline_amd import ops
    gen = torch.Generator().manual_seed(C)
    x, g = torch.randn(1, C, generator=gen).to(dtype).cuda(), (1 + torch.rand(1, C, generator=gen)).to(dtype).cuda()
    _, mean, rstd = ops.layernorm_fwd(x)
    _, _, dbeta = ops.layernorm_bwd(g.expand(M, C), x.expand(M, C), mean.expand(M).contiguous(), rstd.expand(M).contiguous())
    want = (M * g.double())[0]
    assert ((dbeta.double() - want).abs() <= 2 * U * want * (1 + U)).all(), ((dbeta.double() - want).abs() / want).max() / U
