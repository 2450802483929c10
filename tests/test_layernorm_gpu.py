"""Layer norm (csrc/layernorm.hip) against its definition in float64.

Tolerances.  u = 2^-24 is the rounding of a float32 operation, h = torch.finfo(t).eps / 2 the one of the output's type (bf16 2^-8, f16 2^-11).  A thread adds at most 32 elements of a row (a long row: C / 256), the join adds 8 more: at most n = 40 + C / 256 additions, so
  |mean - ref| <= n u max|x|,  xh is off by at most ((n + 2) u max|x|) / sd + (n + 8) u |xh|,  sd = sqrt(var + eps),
and y by |gamma| times that, the rounding of the last multiply-add and its own rounding h |y|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def half(t):
    return torch.finfo(t).eps / 2


def rows_of(M, C, dtype, seed, offset=0.5, layout="dense"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, C, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset).to(dtype)
    return place(x, layout)


def place(x, layout):
    """the same values on the GPU: dense, as columns of a wider 16-byte aligned matrix, at an odd element offset, or every second row"""
    M, C = x.shape
    if layout == "dense":
        return x.cuda()
    if layout == "slab":
        w = torch.full((M, (C + 7) // 8 * 8 + 16), float("nan"), dtype=x.dtype)
        w[:, 8:8 + C] = x
        return w.cuda()[:, 8:8 + C]
    if layout == "odd":
        w = torch.full((M * C + 3,), float("nan"), dtype=x.dtype)
        w[3:] = x.reshape(-1)
        return w.cuda()[3:].view(M, C)
    w = torch.full((2 * M, C), float("nan"), dtype=x.dtype)
    w[::2] = x
    return w.cuda()[::2]


def fwd_ref(x, gamma, beta):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    sd = (var + EPS).sqrt()
    xh = (x - mean) / sd
    y = xh * (gamma.double() if gamma is not None else 1) + (beta.double() if beta is not None else 0)
    return y, mean[:, 0], sd[:, 0], xh


def check_fwd(x, gamma, beta, y, mean, rstd):
    ref, rm, sd, xh = fwd_ref(x, gamma, beta)
    C = x.shape[1]
    n = 40 + C / 256
    top = x.double().abs().amax(1)
    gm = gamma.double().abs() if gamma is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    off = ((n + 2) * U * top / sd)[:, None] + (n + 8) * U * xh.abs()
    bound = gm * off + 2 * U * ref.abs() + 2 * U * (gm * xh.abs()) + half(y.dtype) * ref.abs() + 2.0 ** -24 * (y.dtype == torch.float16)
    assert y.shape == x.shape and y.dtype == x.dtype
    assert ((y.double() - ref).abs() <= bound).all(), ((y.double() - ref).abs() / bound).max()
    assert ((mean.double() - rm).abs() <= (n * U * top) + 1e-40).all()
    # d(var) <= 2 |xh sd| dmean + ..., relative to var + eps: at most (2 n u top / sd + (n + 6) u); rstd half of that and two roundings
    assert ((rstd.double() * sd - 1).abs() <= 2 * n * U * top / sd + (n + 8) * U).all()


SHAPES = [(1, 1), (1, 1280), (3, 7), (17, 128), (16, 8), (37, 144), (5, 256), (65, 257), (9, 512), (11, 1000), (2351, 1001), (7, 2048), (6, 2056), (6, 4096),
          (3, 4104), (2, 8192), (3, 8193), (2, 20000), (5000, 24)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,C", SHAPES)
def test_forward(device, M, C, dtype):
    from speedplusbaseline_amd import ops
    x = rows_of(M, C, dtype, M + C)
    g = torch.Generator().manual_seed(1)
    gamma, beta = (1 + 0.2 * torch.randn(C, generator=g)).cuda(), (0.2 * torch.randn(C, generator=g)).cuda()
    check_fwd(x, gamma, beta, *ops.layernorm_fwd(x, gamma, beta, eps=EPS))


@pytest.mark.parametrize("layout", ["slab", "odd", "second"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,C", [(1, 8), (19, 144), (5, 333), (6, 1024), (3, 4096), (2, 8200)])
def test_forward_strides_without_parameters(device, M, C, dtype, layout):
    from speedplusbaseline_amd import ops
    x = rows_of(M, C, dtype, C, layout=layout)
    check_fwd(x, None, None, *ops.layernorm_fwd(x, eps=EPS))
    out = rows_of(M, C, dtype, 3, layout=layout)
    y, mean, rstd = ops.layernorm_fwd(x, eps=EPS, Y=out)
    assert y.data_ptr() == out.data_ptr()
    check_fwd(x, None, None, y, mean, rstd)
    if layout == "second":                       # the rows between are left as they were
        whole = out.as_strided((2 * M, C), (C, 1))
        assert torch.isnan(whole[1::2]).all()


def test_forward_large_mean_constant_rows_and_nonfinite(device):
    from speedplusbaseline_amd import ops
    for C in (24, 144, 1000, 4096):
        x = rows_of(6, C, torch.float32, C)
        x[0] += 1e4                              # a mean far larger than the spread
        x[1] = 3.25                              # no spread at all
        x[2] = 0
        x[3, C // 2] = float("inf")
        x[4, C - 1] = float("nan")
        keep = [0, 1, 2, 5]
        y, mean, rstd = ops.layernorm_fwd(x, eps=EPS)
        assert torch.isnan(y[3]).any() and torch.isnan(y[4]).all()
        check_fwd(x[keep], None, None, y[keep], mean[keep], rstd[keep])


def test_forward_in_place_broadcast_rows_and_empty(device):
    from speedplusbaseline_amd import ops
    x = rows_of(77, 320, torch.bfloat16, 5)
    want = ops.layernorm_fwd(x)[0]
    y, _, _ = ops.layernorm_fwd(x, Y=x)
    assert y is x and torch.equal(x, want)
    one = rows_of(1, 256, torch.bfloat16, 6)
    y, mean, _ = ops.layernorm_fwd(one.expand(9, 256))
    assert torch.equal(y, ops.layernorm_fwd(one)[0].expand(9, 256)) and mean.shape == (9,)
    y, mean, rstd = ops.layernorm_fwd(torch.empty(0, 16, device="cuda"))
    assert y.shape == (0, 16) and mean.numel() == 0


def bwd_ref(g, x, mean, rstd, gamma):
    g, x, mean, rstd = g.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    gm = gamma.double() if gamma is not None else torch.ones(x.shape[1], dtype=torch.float64, device=x.device)
    xh = (x - mean) * rstd
    h = g * gm
    return rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True)), g * xh, xh, h


def check_bwd(g, x, mean, rstd, gamma, dx, dgamma, dbeta, before=(0, 0)):
    ref, gx, xh, h = bwd_ref(g, x, mean, rstd, gamma)
    M, C = x.shape
    n = 44 + C / 256
    r = rstd.double()[:, None]
    top = x.double().abs().amax(1, keepdim=True) + mean.double().abs()[:, None]
    dxh = 2 * U * xh.abs() + U * top * r                     # rounding of x - mean and of the product
    # sums: n roundings of the sum of magnitudes; a term h xh carries dxh and two roundings
    s1, s2 = h.mean(1, keepdim=True).abs(), (h * xh).mean(1, keepdim=True).abs()
    e1 = n * U * h.abs().mean(1, keepdim=True)
    e2 = n * U * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * dxh).mean(1, keepdim=True)
    bound = r * (4 * U * (h.abs() + s1 + xh.abs() * s2) + e1 + xh.abs() * e2 + dxh * s2) + half(dx.dtype) * ref.abs() + 2.0 ** -24 * (dx.dtype == torch.float16)
    assert ((dx.double() - ref).abs() <= bound).all(), ((dx.double() - ref).abs() / bound).max()
    # a thread adds its rows (at most M / 512 + 1), a workgroup joins 16 groups, the last launch a quarter of at most 512 partial rows and 4 quarters
    k = M / 512 + 1 + 16 + 128 + 8
    for got, terms, extra, b in ((dgamma, gx, (g.double().abs() * dxh).sum(0), before[0]), (dbeta, g.double(), 0, before[1])):
        want = terms.sum(0) + b
        lim = k * U * terms.abs().sum(0) + extra + U * want.abs() + 1e-40
        assert ((got.double() - want).abs() <= lim).all(), ((got.double() - want).abs() / lim).max()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,C", SHAPES)
def test_backward(device, M, C, dtype):
    from speedplusbaseline_amd import ops
    x, g = rows_of(M, C, dtype, M + C), rows_of(M, C, dtype, 7 * M + C, offset=0.0)
    gamma = (1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(1))).cuda()
    _, mean, rstd = ops.layernorm_fwd(x, gamma, eps=EPS)
    check_bwd(g, x, mean, rstd, gamma, *ops.layernorm_bwd(g, x, mean, rstd, gamma))


@pytest.mark.parametrize("layout", ["slab", "odd", "second"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,C", [(1, 8), (19, 144), (5, 333), (700, 1024), (3, 4096), (2, 8200)])
def test_backward_strides_accumulation_and_no_parameters(device, M, C, dtype, layout):
    from speedplusbaseline_amd import ops
    x, g = rows_of(M, C, dtype, C, layout=layout), rows_of(M, C, dtype, C + 1, offset=0.0, layout=layout)
    _, mean, rstd = ops.layernorm_fwd(x, eps=EPS)
    dgamma, dbeta = torch.randn(C, device="cuda"), torch.randn(C, device="cuda")
    before = (dgamma.double(), dbeta.double())
    out = ops.layernorm_bwd(g, x, mean, rstd, None, dgamma, dbeta)
    assert out[1] is dgamma and out[2] is dbeta
    check_bwd(g, x, mean, rstd, None, *out, before=before)
    alone = ops.layernorm_bwd(g, x, mean, rstd, None, param_grads=False)
    assert alone[1] is None and alone[2] is None and torch.equal(alone[0], out[0])
    inplace = ops.layernorm_bwd(g, x, mean, rstd, None, dX=g)          # dX over G: the sums come from the values before
    assert torch.equal(inplace[0], out[0])
    # the same sums, one of them added to what was there: a rounding of the result
    assert ((inplace[1].double() + before[0] - dgamma.double()).abs() <= U * dgamma.double().abs() + 1e-40).all()


def test_backward_against_differences(device):
    """dL/dx, dL/dgamma, dL/dbeta of L = sum(w * y) against central differences of the float64 definition"""
    from speedplusbaseline_amd import ops
    M, C, d = 3, 20, 1e-5
    x, w = rows_of(M, C, torch.float32, 3), rows_of(M, C, torch.float32, 4, offset=0.0)
    gamma, beta = torch.linspace(0.5, 1.5, C).cuda(), torch.linspace(-1, 1, C).cuda()
    _, mean, rstd = ops.layernorm_fwd(x, gamma, beta, eps=EPS)
    dx, dg, db = ops.layernorm_bwd(w, x, mean, rstd, gamma)
    loss = lambda a, b, c: (w.double() * fwd_ref(a, b, c)[0]).sum()          # noqa: E731

    def diff(args, which):
        out = torch.zeros_like(args[which], dtype=torch.float64).reshape(-1)
        for i in range(out.numel()):
            v = [a.double().clone() for a in args]
            v[which].reshape(-1)[i] += d
            up = loss(*v)
            v[which].reshape(-1)[i] -= 2 * d
            out[i] = (up - loss(*v)) / (2 * d)
        return out.view(args[which].shape)
    args = (x, gamma, beta)
    # central differences: d^2 / 6 times a third derivative of a few units, and 2^-53 |L| / d; far below 1e-5, as is the float32 arithmetic
    for got, which in ((dx, 0), (dg, 1), (db, 2)):
        assert ((got.double() - diff(args, which)).abs() <= 1e-5 * (1 + got.double().abs())).all()


def test_backward_empty_and_same_bits_twice(device):
    from speedplusbaseline_amd import ops
    e = torch.empty(0, 40, device="cuda")
    dx, dg, db = ops.layernorm_bwd(e, e, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"))
    assert dx.shape == (0, 40) and (dg == 0).all() and (db == 0).all()
    acc = torch.ones(40, device="cuda"), torch.ones(40, device="cuda")
    ops.layernorm_bwd(e, e, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), None, *acc)
    assert (acc[0] == 1).all() and (acc[1] == 1).all()
    x, g = rows_of(20000, 96, torch.bfloat16, 1), rows_of(20000, 96, torch.bfloat16, 2)
    _, mean, rstd = ops.layernorm_fwd(x)
    a, b = ops.layernorm_bwd(g, x, mean, rstd), ops.layernorm_bwd(g, x, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_longest_register_rows_behind_two_to_the_32(device):
    """more than 2^32 bytes in front of the last rows"""
    from speedplusbaseline_amd import ops
    M, C = 300000, 8192                                     # 4.9 GB of bfloat16
    x = torch.zeros(M, C, dtype=torch.bfloat16, device="cuda")
    tail = rows_of(4, C, torch.bfloat16, 9)
    x[-4:] = tail
    y, mean, rstd = ops.layernorm_fwd(x)
    assert torch.equal(y[-4:], ops.layernorm_fwd(tail)[0]) and (y[1000] == 0).all()
    dx, dg, db = ops.layernorm_bwd(x, x, mean, rstd, dX=y)
    want = ops.layernorm_bwd(tail, tail, mean[-4:].contiguous(), rstd[-4:].contiguous())
    assert torch.equal(dx[-4:], want[0]) and torch.allclose(db, want[2], rtol=1e-6, atol=1e-6)


def test_rows_behind_two_to_the_32(device):
    """2.6e9 elements in place: the last rows as in a call of their own, forward and backward"""
    from speedplusbaseline_amd import ops
    M, C, last = 640000, 4096, 64
    tail, g = rows_of(last, C, torch.bfloat16, 1), rows_of(last, C, torch.bfloat16, 2)
    gamma = torch.randn(C, device="cuda")
    want, mean, rstd = ops.layernorm_fwd(tail, gamma)
    dx, dg, db = ops.layernorm_bwd(g, tail, mean, rstd, gamma)
    X = torch.zeros(M, C, dtype=torch.bfloat16, device="cuda")
    X[-last:] = tail
    G = torch.zeros_like(X)
    G[-last:] = g
    y, m, r = ops.layernorm_fwd(X, gamma)
    assert torch.equal(y[-last:], want) and torch.equal(m[-last:], mean) and torch.equal(r[-last:], rstd) and (y[:last] == 0).all()
    d, dgamma, dbeta = ops.layernorm_bwd(G, X, m, r, gamma, dX=G)
    assert torch.equal(d[-last:], dx) and (d[:last] == 0).all()
    # the sums over rows: the same 64 terms in another order
    top = lambda t: 70 * U * t.abs().sum(0)
    xh = (tail.double() - mean.double()[:, None]) * rstd.double()[:, None]
    assert ((dgamma.double() - dg.double()).abs() <= top(g.double() * xh) * 2).all() and ((dbeta.double() - db.double()).abs() <= top(g.double()) * 2).all()
