"""What layer norm and the 8-bit operators refuse, at the C entries (before anything touches a device) and in speedplusbaseline_amd.ops."""
import ctypes as C

import pytest
import torch

from speedplusbaseline_amd import _args8 as A8, _lib as L, ops

ARG, SHAPE = -1, -2
P16 = C.c_void_p(1 << 20)       # an aligned address that is never read
ODD = C.c_void_p((1 << 20) + 1)


def norm(**kw):
    a = A8.LayerNormArgs()
    for k in ("X", "G", "Y", "mean", "rstd", "dgamma", "dbeta", "part"):
        setattr(a, k, P16)
    a.M, a.C, a.ldx, a.ldg, a.ldy, a.eps, a.part_cap = 4, 32, 32, 32, 32, 1e-5, 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


@pytest.mark.parametrize("lib", [L.lib, L.lib_f16], ids=["bf16", "f16"])
def test_layernorm_refusals(lib):
    l = lib()
    for fn in (l.spb_layernorm_fwd, l.spb_layernorm_bwd):
        assert fn(2, norm(), None) == ARG and fn(-1, norm(), None) == ARG and fn(0, None, None) == ARG
        for kw in (dict(C=0), dict(C=-3), dict(M=-1), dict(ldx=-1), dict(ldy=31)):
            assert fn(0, norm(**kw), None) == SHAPE, kw
        for k in ("X", "Y", "mean", "rstd"):
            assert fn(1, norm(**{k: None}), None) == ARG, k
    assert l.spb_layernorm_bwd(1, norm(G=None), None) == ARG
    assert l.spb_layernorm_bwd(1, norm(ldg=-2), None) == SHAPE
    assert l.spb_layernorm_bwd(1, norm(part=None), None) == ARG
    assert l.spb_layernorm_bwd(1, norm(part_cap=l.spb_layernorm_bwd_floats(4, 32) - 1), None) == ARG
    assert l.spb_layernorm_fwd(1, norm(M=0, X=None), None) == 0
    assert l.spb_layernorm_bwd_floats(-1, 8) == SHAPE and l.spb_layernorm_bwd_floats(8, 0) == SHAPE and l.spb_layernorm_bwd_floats(0, 8) > 0


@pytest.mark.parametrize("lib", [L.lib, L.lib_f16], ids=["bf16", "f16"])
def test_packing_refusals(lib):
    l = lib()
    rows = lambda dt=1, X=P16, ld=128, M=4, K=128, q=P16, s=P16: l.spb_pack8_rows(dt, X, ld, M, K, q, s, None)                    # noqa: E731
    assert rows(dt=2) == ARG and rows(X=None) == ARG and rows(q=None) == ARG and rows(s=None) == ARG and rows(q=ODD) == ARG and rows(s=ODD) == ARG
    assert rows(M=-1) == SHAPE and rows(K=-1) == SHAPE and rows(ld=-1) == SHAPE and rows(M=0, X=None) == 0 and rows(K=0, X=None) == 0
    assert rows(M=1 << 32, K=128) == SHAPE
    w = lambda dt=1, W=P16, ld=128, N=4, K=128, q=P16, s=P16, qt=P16, st=P16: l.spb_pack8_weight(dt, W, ld, N, K, q, s, qt, st, None)   # noqa: E731
    assert w(dt=5) == ARG and w(W=None) == ARG and w(qt=None) == ARG and w(st=None) == ARG and w(qt=ODD) == ARG and w(N=-1) == SHAPE and w(ld=-1) == SHAPE
    u = lambda dt=1, q=P16, s=P16, br=1, M=4, K=128, Y=P16, ld=128: l.spb_unpack8(dt, q, s, br, M, K, Y, ld, None)                 # noqa: E731
    assert u(dt=9) == ARG and u(br=2) == ARG and u(Y=None) == ARG and u(q=ODD) == ARG and u(ld=127) == SHAPE and u(M=-1) == SHAPE and u(M=0) == 0
    f = lambda dt=1, act=4, X=P16, Y=P16, ldx=128, ldy=128, M=4, K=128, q=P16, s=P16: l.spb_act8_fwd(dt, act, X, ldx, Y, ldy, M, K, q, s, None)   # noqa: E731
    assert f(act=3) == ARG and f(act=7) == ARG and f(act=0) == ARG and f(X=None) == ARG and f(Y=None) == ARG and f(q=None) == ARG and f(ldy=5) == SHAPE and f(K=0) == 0
    b = lambda dt=1, act=4, G=P16, D=P16, ldg=128, ldd=128, M=4, K=128, q=P16, s=P16: l.spb_act8_bwd(dt, act, G, ldg, q, s, D, ldd, M, K, None)   # noqa: E731
    assert b(act=2) == ARG and b(G=None) == ARG and b(D=None) == ARG and b(s=None) == ARG and b(ldd=5) == SHAPE and b(ldg=-1) == SHAPE and b(M=0) == 0


def product(**kw):
    a = A8.Gemm8Args()
    for k in ("A", "As", "B", "Bs", "Y", "ws"):
        setattr(a, k, P16)
    a.M, a.N, a.K, a.ldy, a.b_block_rows, a.ws_bytes = 4, 64, 256, 64, 128, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def wgrad(**kw):
    a = A8.Wgrad8Args()
    for k in ("G", "X", "Xs", "dW", "ws"):
        setattr(a, k, P16)
    a.M, a.N, a.K, a.ldg, a.ldw, a.ws_bytes = 100000, 64, 256, 64, 256, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


@pytest.mark.parametrize("lib", [L.lib, L.lib_f16], ids=["bf16", "f16"])
def test_product_refusals(lib):
    l = lib()
    assert l.spb_gemm8(3, product(), None) == ARG and l.spb_gemm8(1, None, None) == ARG and l.spb_gemm8(1, product(b_block_rows=64), None) == ARG
    for kw in (dict(M=-1), dict(N=-1), dict(K=-1), dict(ldy=63), dict(K=(1 << 23) + 1)):
        assert l.spb_gemm8(1, product(**kw), None) == SHAPE, kw
    for k in ("A", "As", "B", "Bs", "Y"):
        assert l.spb_gemm8(1, product(**{k: None}), None) == ARG, k
    for k in ("A", "As", "B", "Bs"):
        assert l.spb_gemm8(1, product(**{k: ODD}), None) == ARG, k
    assert l.spb_gemm8(1, product(M=0, A=None), None) == 0 and l.spb_gemm8(1, product(N=0, A=None), None) == 0
    for dt in (0, 1):
        for M, N, K in ((1, 64, 100000), (1000, 16, 50000), (64, 64, 64)):
            need = l.spb_gemm8_bytes(dt, M, N, K)
            assert need >= 0
            if need:
                assert l.spb_gemm8(dt, product(M=M, N=N, K=K, ws_bytes=need - 1), None) == ARG
                assert l.spb_gemm8(dt, product(M=M, N=N, K=K, ws=None), None) == ARG
    assert l.spb_gemm8_bytes(4, 1, 1, 1) < 0 and l.spb_gemm8_bytes(1, -1, 1, 1) < 0
    assert l.spb_gemm8_wgrad(2, wgrad(), None) == ARG and l.spb_gemm8_wgrad(1, None, None) == ARG
    for kw in (dict(M=-1), dict(N=-1), dict(K=-1), dict(ldg=-1), dict(ldw=255), dict(K=(1 << 23) + 1)):
        assert l.spb_gemm8_wgrad(1, wgrad(**kw), None) == SHAPE, kw
    for kw in (dict(G=None), dict(X=None), dict(Xs=None), dict(dW=None), dict(X=ODD), dict(Xs=ODD), dict(ws=None), dict(ws=ODD),
               dict(ws_bytes=l.spb_gemm8_wgrad_bytes(1, 100000, 64, 256) - 1)):
        assert l.spb_gemm8_wgrad(1, wgrad(**kw), None) == ARG, kw
    assert l.spb_gemm8_wgrad(1, wgrad(N=0, G=None), None) == 0
    assert l.spb_gemm8_wgrad_bytes(1, 100000, 64, 256) > 0 and l.spb_gemm8_wgrad_bytes(1, 0, 64, 256) == 0 and l.spb_gemm8_wgrad_bytes(7, 1, 1, 1) < 0


@pytest.mark.parametrize("lib", [L.lib, L.lib_f16], ids=["bf16", "f16"])
def test_products_refuse_sides_that_do_not_fit_their_offsets(lib):
    l, deep, wide = lib(), (1 << 23) + 1, (1 << 30) + 1
    assert l.spb_gemm8(1, product(N=wide, ldy=wide), None) == SHAPE and l.spb_gemm8_wgrad(1, wgrad(N=wide, ldg=wide), None) == SHAPE
    for f in (l.spb_gemm8_bytes, l.spb_gemm8_wgrad_bytes):
        assert f(1, 100, wide, 128) == SHAPE and f(1, 100, 128, deep) == SHAPE and f(1, 100, wide - 1, 128) >= 0 and f(1, 100, 128, deep - 1) >= 0


def test_argument_structs_have_the_layout_of_the_header(tmp_path):
    import os
    import subprocess
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "spb_hip.h"', 'int main(void) {']
    for py, c in (("LayerNormArgs", "spb_layernorm_args_t"), ("Gemm8Args", "spb_gemm8_args_t"), ("Wgrad8Args", "spb_wgrad8_args_t")):
        src.append('printf("%s sizeof %%zu\\n", sizeof(%s));' % (py, c))
        src += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (py, f[0], c, f[0]) for f in getattr(A8, py)._fields_]
    (tmp_path / "abi.c").write_text("\n".join(src + ['printf("act x %d%d%d\\n", SPB_ACT_GELU, SPB_ACT_GELU_TANH, SPB_ACT_SILU);', 'return 0; }']))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "abi.c"), "-o", str(tmp_path / "abi")], check=True)
    for line in subprocess.run([str(tmp_path / "abi")], capture_output=True, text=True, check=True).stdout.splitlines():
        py, name, val = line.split()
        if py == "act":
            assert val == "%d%d%d" % (L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU)
            continue
        cls = getattr(A8, py)
        assert int(val) == (C.sizeof(cls) if name == "sizeof" else getattr(cls, name).offset), line


def test_ops_refuse_host_tensors():
    x = torch.zeros(4, 8)
    P = ops.Packed8.empty(4, 8, 1, "cpu")
    for call in (lambda: ops.layernorm_fwd(x), lambda: ops.layernorm_bwd(x, x, x[:, 0], x[:, 0]), lambda: ops.quant8(x), lambda: ops.quant8_weight(x),
                 lambda: ops.dequant8(P), lambda: ops.gemm8(P, P), lambda: ops.gemm8_wgrad(x, P), lambda: ops.act8_fwd(x, L.ACT_GELU), lambda: ops.act8_bwd(x, P, L.ACT_GELU),
                 lambda: ops.act8_fwd(x, L.ACT_RELU), lambda: ops.gemm8(x, P)):
        with pytest.raises(RuntimeError):
            call()
