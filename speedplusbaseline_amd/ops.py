"""Thin torch-tensor front end of the per-kernel C-ABI entry points (used by the parity tests and by callers that
want a single fused op).  Tensors are device memory only; all arithmetic happens in libspb_hip.so.
"""
import ctypes as C

import torch

from . import _args8 as A8
from . import _lib as L

_DT = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.BF16}   # float16: the same 16-bit code, served by the IEEE-half twin library


def lib_of(t):
    """the library that understands tensor t's 16-bit format: libspb_hip_f16.so for float16, libspb_hip.so otherwise"""
    return L.lib_f16() if (t is not None and t.dtype == torch.float16) else L.lib()


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("speedplusbaseline_amd ops run on the GPU only (got a %s tensor)" % t.device)
        if t is not None and not t.is_contiguous():
            raise RuntimeError("speedplusbaseline_amd ops need contiguous tensors")


def _need_rows(*ts):
    """2-D operands that may be column slabs of a wider row-major matrix (unit column stride, any row stride)"""
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("speedplusbaseline_amd ops run on the GPU only (got a %s tensor)" % t.device)
        if t.dim() != 2 or t.stride(1) != 1 or (t.stride(0) & 7) or (t.storage_offset() & 7):
            raise RuntimeError("speedplusbaseline_amd GEMM operands are row-major 2-D tensors or 8-aligned column slabs of one")


def dtype_code(t, twin=False):
    """16-bit / 32-bit code of tensor t for the C-ABI.  float16 shares bfloat16's code and is only meaningful in the IEEE-half
    twin library (lib_of): entry points that exist in libspb_hip.so alone (the KRN kernels) pass twin=False and refuse it
    instead of reading half bits as bfloat16."""
    if t.dtype == torch.float16 and not twin:
        raise RuntimeError("this kernel has no float16 instance (bfloat16 / float32 only): float16 is built for the SPN path "
                           "(libspb_hip_f16.so); KRN / RevGrad use --precision bf16")
    try:
        return _DT[t.dtype]
    except KeyError:
        raise RuntimeError("activation dtype must be float32, bfloat16 or float16, got %s" % t.dtype)


def bnref(C_, sums=None, gamma=None, beta=None, bsums=None, n=1, R=1, act=L.ACT_NONE, slope=0.0, eps=1e-5, moments=0):
    """spb_bnref_t from f32 tensors. gamma=None means identity (already normalised tensor)."""
    _need_cuda(sums, gamma, beta, bsums)
    r = L.BNRef()
    r.sums = _ptr(sums); r.gamma = _ptr(gamma); r.beta = _ptr(beta); r.bsums = _ptr(bsums)
    r.inv_n = 1.0 / float(n); r.eps = eps; r.slope = slope; r.C = C_; r.R = R; r.act = act; r.moments = moments
    r._keep = (sums, gamma, beta, bsums)
    return r


def pwconv_gemm(A, Bw, Y, pro, pro_mode, epi_mode, A2=None, res=None, Zout=None, bias=None, osums=None, epi=None,
                out_act=L.ACT_NONE, oR=1, out_scale=1.0, pro2=None, Ymat=None):
    if Y is None:               # statistics only (epi_mode 1): the batch sums of a product that is never stored
        _need_rows(A)
    else:
        _need_rows(A, Y)
    _need_cuda(Bw, A2, res, Zout, bias, osums)
    g = L.GemmArgs()
    g.A = _ptr(A); g.A2 = _ptr(A2); g.Bw = _ptr(Bw); g.Y = _ptr(Y); g.res = _ptr(res); g.Zout = _ptr(Zout)
    g.bias = _ptr(bias); g.osums = _ptr(osums); g.pro = pro
    g.epi = epi if epi is not None else bnref(Bw.shape[0])
    g.M, g.K = A.shape[0], A.shape[1]; g.N = Bw.shape[0]
    g.lda = A.stride(0) if A.stride(0) != A.shape[1] else 0     # column slabs of wider matrices (grouped convolutions)
    g.ldc = 0 if Y is None else (Y.stride(0) if Y.stride(0) != Y.shape[1] else 0)
    g.pro_mode = pro_mode; g.epi_mode = epi_mode; g.out_act = out_act; g.oR = oR; g.out_scale = out_scale
    if pro_mode == 3:       # residual join: a = bn(A) + bn2(A2), written to Ymat by the launch
        _need_cuda(Ymat)
        g.pro2 = pro2 if pro2 is not None else bnref(A.shape[1]); g.Ymat = _ptr(Ymat)
    elif Ymat is not None:  # statistics-only pass (Y is None): also write the operand round16(act(bn(A)))
        _need_cuda(Ymat)
        g.Ymat = _ptr(Ymat)
    L.check(lib_of(A).spb_pwconv_gemm(dtype_code(A, True), C.byref(g), _stream()), "spb_pwconv_gemm")


def pwconv_wgrad(G, X, dW, pro_dz, pro_a, Zn=None):
    _need_rows(G, X)
    _need_cuda(dW, Zn)
    w = L.WgradArgs()
    w.G = _ptr(G); w.Zn = _ptr(Zn); w.X = _ptr(X); w.dW = _ptr(dW); w.pro_dz = pro_dz; w.pro_a = pro_a
    w.M = G.shape[0]; w.N = G.shape[1]; w.K = X.shape[1]
    w.ldg = G.stride(0) if G.stride(0) != G.shape[1] else 0
    w.ldx = X.stride(0) if X.stride(0) != X.shape[1] else 0
    L.check(lib_of(G).spb_pwconv_wgrad(dtype_code(G, True), C.byref(w), _stream()), "spb_pwconv_wgrad")


def pwconv_bwd_fused(G, Zn, Wt, X, Zout, Y, dW, osums, pro_dz, pro_a, epi, res=None, oR=1):
    """Fused input-gradient + weight-gradient of a pointwise conv.  Returns False when the library has no fused instance
    for this (dtype, N, K) -- the caller then uses pwconv_gemm + pwconv_wgrad."""
    _need_cuda(G, Zn, Wt, X, Zout, Y, dW, osums, res)
    a = L.PwBwdArgs()
    a.G = _ptr(G); a.Zn = _ptr(Zn); a.Wt = _ptr(Wt); a.X = _ptr(X); a.Zout = _ptr(Zout); a.res = _ptr(res); a.Y = _ptr(Y)
    a.dW = _ptr(dW); a.osums = _ptr(osums); a.pro_dz = pro_dz; a.pro_a = pro_a; a.epi = epi
    a.M = G.shape[0]; a.N = G.shape[1]; a.K = X.shape[1]; a.oR = oR
    code = L.lib().spb_pwconv_bwd_fused(dtype_code(G), C.byref(a), _stream())
    if code == -4:  # SPB_E_UNSUPPORTED
        return False
    L.check(code, "spb_pwconv_bwd_fused")
    return True


def _dwargs(X, Wd, B, H, W_, C_, stride, **kw):
    d = L.DwArgs()
    d.X = _ptr(X); d.Wd = _ptr(Wd); d.B = B; d.H = H; d.W = W_; d.C = C_; d.stride = stride
    for k, v in kw.items():
        if isinstance(v, torch.Tensor) or v is None:
            setattr(d, k, _ptr(v))
        else:
            setattr(d, k, v)
    ident = bnref(C_)
    for k in ("pro", "pro_in", "epi"):
        if k not in kw or kw[k] is None:
            setattr(d, k, ident)
    if "oR" not in kw:
        d.oR = 1
    d.xe = bnref(8)
    return d


def _set_expand(d, expand):
    """spb_dw_args_t::Xe -- the depthwise layer's input is the (never stored) output of a 1x1 expand convolution:
    expand = (Xe [B,H,W,Ce], We [C,Ce] compute dtype, xe = BN/activation turning Xe into that convolution's operand or None)"""
    Xe, We, xe = expand
    _need_cuda(Xe, We)
    d.Xe = _ptr(Xe); d.We = _ptr(We); d.Ce = Xe.shape[-1]
    d.xe = xe if xe is not None else bnref(Xe.shape[-1])
    d._keep_expand = (Xe, We, xe)


def dwconv_fwd(X, Wd, Y, pro, stride, osums=None, oR=1, expand=None):
    """expand: see _set_expand; X is then None and `pro` names the BatchNorm / activation on the recomputed tensor"""
    src = X if expand is None else expand[0]
    B, H, W_ = src.shape[:3]
    C_ = Y.shape[3]
    _need_cuda(X, Wd, Y, osums)
    d = _dwargs(X, Wd, B, H, W_, C_, stride, Y=Y, pro=pro, osums=osums, oR=oR, epi_mode=1 if osums is not None else 0)
    if expand is not None:
        _set_expand(d, expand)
    L.check(L.lib().spb_dwconv_fwd(dtype_code(Y), C.byref(d), _stream()), "spb_dwconv_fwd")


def dwconv_dgrad(G, Z, Wd, Y, pro, stride, in_hw, epi=None, Zout=None, res=None, osums=None, oR=1, dW=None, Xin=None,
                 pro_in=None, entry_flag=None, entry_val=0, expand=None):
    """Input gradient of the depthwise conv.  With `dW` the weight gradient is accumulated in the same pass; `Xin` and
    `pro_in` (the conv's input tensor and its BN/activation) are then required unless `epi`/`Zout` already name them.
    `entry_flag` (a device int32 word): the launch's first thread stores `entry_val` there before anything else
    (spb_dw_args_t::entry_flag: a stream fork without an event)."""
    B, C_ = G.shape[0], G.shape[3]
    _need_cuda(G, Z, Wd, Y, Zout, res, osums, dW, Xin)
    kw = dict(X2=Z, Y=Y, pro=pro, epi_mode=2 if epi is not None else 0, oR=oR)
    if epi is not None:
        kw.update(epi=epi, Zout=Zout, res=res, osums=osums)
    if dW is not None:
        kw.update(dW=dW)
        if epi is None:
            kw.update(epi=pro_in, Zout=Xin)
    d = _dwargs(G, Wd, B, in_hw[0], in_hw[1], C_, stride, **kw)
    if entry_flag is not None:
        _need_cuda(entry_flag)
        d.entry_flag = _ptr(entry_flag); d.entry_val = int(entry_val)
    if expand is not None:      # the conv input (Zout / Xin) is recomputed: `epi` / `pro_in` name the BatchNorm on the recomputed tensor
        _set_expand(d, expand)
    L.check(L.lib().spb_dwconv_dgrad(dtype_code(G), C.byref(d), _stream()), "spb_dwconv_dgrad")


def dwconv_wgrad(G, Z, Xin, Wd, dW, pro, pro_in, stride, expand=None):
    src = Xin if expand is None else expand[0]
    B, H, W_ = src.shape[:3]
    C_ = G.shape[3]
    _need_cuda(G, Z, Xin, Wd, dW)
    d = _dwargs(G, Wd, B, H, W_, C_, stride, X2=Z, Xin=Xin, dW=dW, pro=pro, pro_in=pro_in)
    if expand is not None:
        _set_expand(d, expand)
    L.check(L.lib().spb_dwconv_wgrad(dtype_code(G), C.byref(d), _stream()), "spb_dwconv_wgrad")


def stem_fwd(x_nchw, w, y_nhwc, osums=None, oR=1):
    _need_cuda(x_nchw, w, y_nhwc, osums)
    B, _, H, W_ = x_nchw.shape
    L.check(L.lib().spb_stem_fwd(dtype_code(y_nhwc), _ptr(x_nchw), _ptr(w), _ptr(y_nhwc), _ptr(osums), oR, B, H, W_,
                                 _stream()), "spb_stem_fwd")


def stem_wgrad(x_nchw, G, Z, pro_dz, dW):
    _need_cuda(x_nchw, G, Z, dW)
    B, _, H, W_ = x_nchw.shape
    L.check(L.lib().spb_stem_wgrad(dtype_code(G), _ptr(x_nchw), _ptr(G), _ptr(Z), C.byref(pro_dz), _ptr(dW), B, H, W_,
                                   _stream()), "spb_stem_wgrad")


def bn_apply(Z, Y, bn, res=None, bn_res=None, ldc=None, coff=0, reorg=0):
    _need_cuda(Z, Y, res)
    B, H, W_, C_ = Z.shape
    a = L.BnApplyArgs()
    a.Z = _ptr(Z); a.res = _ptr(res); a.Y = _ptr(Y); a.bn = bn
    a.bn_res = bn_res if bn_res is not None else bnref(C_)
    a.B, a.H, a.W, a.C = B, H, W_, C_
    a.ldc = ldc if ldc is not None else C_
    a.coff = coff; a.reorg = reorg
    L.check(L.lib().spb_bn_apply(dtype_code(Z), C.byref(a), _stream()), "spb_bn_apply")


def bn_bwd_prep(dY, Z, G, osums, bn, ldc=None, coff=0, reorg=0, oR=1):
    _need_cuda(dY, Z, G, osums)
    B, H, W_, C_ = Z.shape
    a = L.BnBwdArgs()
    a.dY = _ptr(dY); a.Z = _ptr(Z); a.G = _ptr(G); a.osums = _ptr(osums); a.bn = bn
    a.B, a.H, a.W, a.C = B, H, W_, C_
    a.ldc = ldc if ldc is not None else C_
    a.coff = coff; a.reorg = reorg; a.oR = oR
    L.check(L.lib().spb_bn_bwd_prep(dtype_code(Z), C.byref(a), _stream()), "spb_bn_bwd_prep")


def head_fwd(Z, Wp, bias, pro, J, HW, C_, target=None, S=256, partial=None):
    """Z [B, HW*C]; Wp [Jp, HW*C] (compute dtype). Returns pred [B,J], scalars [3], dout [B,J].  partial: the reduction workspace
    (S*B*Jp floats, zero before its first use; every call leaves it zero again) -- a fresh one is allocated when None."""
    _need_cuda(Z, Wp, bias, target)
    B = Z.shape[0]
    Jp = Wp.shape[0]
    dev = Z.device
    if partial is None:
        partial = torch.zeros(S * B * Jp, dtype=torch.float32, device=dev)   # ends in the reduction's ticket word: zero before the first call
    pred = torch.empty(B, J, dtype=torch.float32, device=dev)
    dout = torch.zeros(B, J, dtype=torch.float32, device=dev)
    scalars = torch.zeros(3, dtype=torch.float32, device=dev)
    h = L.HeadArgs()
    h.Z = _ptr(Z); h.Wp = _ptr(Wp); h.bias = _ptr(bias); h.target = _ptr(target); h.partial = _ptr(partial)
    h.pred = _ptr(pred); h.dout = _ptr(dout); h.scalars = _ptr(scalars); h.pro = pro
    h.B, h.J, h.Jp, h.HW, h.C, h.S = B, J, Jp, HW, C_, S
    L.check(L.lib().spb_head_fwd(dtype_code(Z), C.byref(h), _stream()), "spb_head_fwd")
    return pred, scalars, dout


def head_bwd(Z, Wp, dout, G, osums, dW, dbias, pro, J, HW, C_, gscale=1.0, oR=1):
    _need_cuda(Z, Wp, dout, G, osums, dW, dbias)
    h = L.HeadBwdArgs()
    h.Z = _ptr(Z); h.Wp = _ptr(Wp); h.dout = _ptr(dout); h.G = _ptr(G); h.osums = _ptr(osums); h.dW = _ptr(dW)
    h.dbias = _ptr(dbias); h.pro = pro; h.gscale = gscale
    h.B, h.J, h.Jp, h.HW, h.C, h.oR = Z.shape[0], J, Wp.shape[0], HW, C_, oR
    L.check(L.lib().spb_head_bwd(dtype_code(Z), C.byref(h), _stream()), "spb_head_bwd")


def grad_sqnorm(grads, out):
    _need_cuda(grads, out)
    L.check(L.lib().spb_grad_sqnorm(_ptr(grads), grads.numel(), _ptr(out), _stream()), "spb_grad_sqnorm")


SQ_PARTS = 256


def grad_sqnorm_partials(grads, out):
    """sum of squares of the arena as SQ_PARTS partial sums (no arrival counter); optim_step(sq_partials=out) adds them up"""
    _need_cuda(grads, out)
    assert out.numel() >= SQ_PARTS and out.dtype == torch.float32
    L.check(L.lib().spb_grad_sqnorm_partials(_ptr(grads), grads.numel(), _ptr(out), _stream()), "spb_grad_sqnorm_partials")


def arena_zero(arena):
    """optimizer.zero_grad() on a flat f32 arena (no ATen kernel on the hot path)"""
    _need_cuda(arena)
    L.check(L.lib().spb_arena_zero(_ptr(arena), arena.numel(), _stream()), "spb_arena_zero")


def arena_add(dst, src):
    _need_cuda(dst, src)
    L.check(L.lib().spb_arena_add(_ptr(dst), _ptr(src), dst.numel(), _stream()), "spb_arena_add")


OPT_KIND = {"sgd": 0, "rmsprop": 1, "adam": 2, "adamw": 3}


def optim_step(kind, params, grads, m=None, v=None, sqnorm=None, gmul=None, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
               weight_decay=0.0, max_norm=0.0, clip_value=0.0, step=1, first_step=False, hyper=None, shadow=None, max_blocks=0,
               sq_partials=None, skip=None):
    a = _optim_args(kind, params, grads, m, v, sqnorm, gmul, lr, beta1, beta2, eps, weight_decay, max_norm, clip_value, step, first_step,
                    hyper, shadow, max_blocks)
    if sq_partials is not None:
        _need_cuda(sq_partials)
        a.sq_partials = _ptr(sq_partials); a.n_sq_partials = SQ_PARTS
    if skip is not None:
        _need_cuda(skip)
        a.skip = _ptr(skip)
    L.check(lib_of(shadow).spb_optim_step(C.byref(a), _stream()), "spb_optim_step")   # a float16 shadow: the half twin writes it


def _optim_args(kind, params, grads, m, v, sqnorm, gmul, lr, beta1, beta2, eps, weight_decay, max_norm, clip_value, step, first_step,
                hyper, shadow, max_blocks):
    _need_cuda(params, grads, m, v, sqnorm, gmul, hyper, shadow)
    a = L.OptimArgs()
    a.params = _ptr(params); a.grads = _ptr(grads); a.m = _ptr(m); a.v = _ptr(v); a.sqnorm = _ptr(sqnorm)
    a.gmul = _ptr(gmul); a.hyper = _ptr(hyper); a.n = params.numel(); a.kind = OPT_KIND[kind]
    a.lr = lr; a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.weight_decay = weight_decay
    a.max_norm = max_norm; a.clip_value = clip_value; a.shadow_bf16 = _ptr(shadow); a.max_blocks = max_blocks
    a.bias_c1 = 1.0 - beta1 ** step; a.bias_c2 = 1.0 - beta2 ** step; a.first_step = 1 if first_step else 0
    return a


def fc_wgrad_update(gT, xT, M, kind, params, grads=None, m=None, v=None, gmul=None, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                    weight_decay=0.0, clip_value=0.0, step=1, first_step=False, shadow=None):
    """weight gradient of a fully connected layer (params: its [N][K] weight) fused with its optimizer step (spb_fc_wgrad_update)"""
    _need_cuda(gT, xT)
    N, K = params.shape
    a = _optim_args(kind, params, grads, m, v, None, gmul, lr, beta1, beta2, eps, weight_decay, 0.0, clip_value, step, first_step, None,
                    shadow, 0)
    L.check(lib_of(gT).spb_fc_wgrad_update(_ptr(gT), _ptr(xT), M, N, K, C.byref(a), _stream()), "spb_fc_wgrad_update")


# ---- layer norm, 8-bit linear layers and checkpoints ---------------------------------------------------------------------------------
# Operands are 2-D with contiguous columns and any row stride.  Like every function of this file they enqueue on the current stream and build no
# autograd graph: the backward pass is the explicit *_bwd / *_wgrad call.  They run on the device of their tensors, whichever is current.

def _call(dev, fn, what, *args):
    if dev.index == torch.cuda.current_device():
        L.check(fn(*args, _stream()), what)
    else:
        with torch.cuda.device(dev):
            L.check(fn(*args, _stream()), what)


def _mat(t, name, dev=None, out=False):
    """2-D operand: device memory, contiguous columns, one of the three types; returns its row stride"""
    if not t.is_cuda:
        raise RuntimeError("speedplusbaseline_amd ops run on the GPU only (got a %s tensor for %s)" % (t.device, name))
    if dev is not None and t.device != dev:
        raise RuntimeError("%s is on %s, the other operands on %s" % (name, t.device, dev))
    if t.dtype not in _DT:
        raise RuntimeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise RuntimeError("%s must be 2-D with contiguous columns, got shape %s, strides %s" % (name, tuple(t.shape), t.stride()))
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if out and ld < t.shape[1]:
        raise RuntimeError("the rows of %s overlap" % name)
    return ld


def _like(t, shape, dtype, name, dev):
    if t.device != dev or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise RuntimeError("%s must be %s %s on %s, got %s %s on %s" % (name, dtype, tuple(shape), dev, t.dtype, tuple(t.shape), t.device))


def _vec(t, n, name, dev):
    """contiguous float32 vector of n elements, or None"""
    if t is None:
        return
    _like(t, (n,), torch.float32, name, dev)
    if not t.is_contiguous():
        raise RuntimeError("%s must be contiguous" % name)


def layernorm_fwd(X, gamma=None, beta=None, eps=1e-5, Y=None):
    """Layer norm over the columns of X [M, C]: returns (Y, mean, rstd); mean and rstd (float32 [M]) are what layernorm_bwd needs.  gamma / beta:
    float32 [C] or None (1 / 0).  Y: optional output of X's type, may be X itself."""
    ldx = _mat(X, "X")
    dev, (M, Cn) = X.device, X.shape
    if Cn < 1:
        raise RuntimeError("layernorm needs at least one column")
    _vec(gamma, Cn, "gamma", dev); _vec(beta, Cn, "beta", dev)
    if Y is None:
        Y = torch.empty(M, Cn, dtype=X.dtype, device=dev)
    else:
        _like(Y, X.shape, X.dtype, "Y", dev)
    stats = torch.empty(2, M, dtype=torch.float32, device=dev)
    mean, rstd = stats[0], stats[1]
    a = A8.LayerNormArgs()
    a.X, a.Y, a.gamma, a.beta, a.mean, a.rstd = _ptr(X), _ptr(Y), _ptr(gamma), _ptr(beta), _ptr(mean), _ptr(rstd)
    a.M, a.C, a.ldx, a.ldy, a.eps = M, Cn, ldx, _mat(Y, "Y", dev, out=True), eps
    _call(dev, lib_of(X).spb_layernorm_fwd, "spb_layernorm_fwd", dtype_code(X, True), C.byref(a))
    return Y, mean, rstd


def layernorm_bwd(G, X, mean, rstd, gamma=None, dgamma=None, dbeta=None, dX=None, param_grads=True):
    """Backward of layernorm_fwd: returns (dX, dgamma, dbeta).  dgamma / dbeta given: accumulated into (both or neither), otherwise new;
    param_grads=False: not computed (None).  dX: optional output, may be G itself."""
    ldg, ldx = _mat(G, "G"), _mat(X, "X", G.device)
    dev, (M, Cn) = X.device, X.shape
    if Cn < 1:
        raise RuntimeError("layernorm needs at least one column")
    _like(G, X.shape, X.dtype, "G", dev)
    _vec(gamma, Cn, "gamma", dev); _vec(mean, M, "mean", dev); _vec(rstd, M, "rstd", dev)
    _vec(dgamma, Cn, "dgamma", dev); _vec(dbeta, Cn, "dbeta", dev)
    if (dgamma is None) != (dbeta is None) or (dgamma is not None and not param_grads):
        raise RuntimeError("dgamma and dbeta are accumulated into together")
    if dX is None:
        dX = torch.empty(M, Cn, dtype=X.dtype, device=dev)
    else:
        _like(dX, X.shape, X.dtype, "dX", dev)
    lib = lib_of(X)
    a = A8.LayerNormArgs()
    a.X, a.G, a.Y, a.gamma, a.mean, a.rstd = _ptr(X), _ptr(G), _ptr(dX), _ptr(gamma), _ptr(mean), _ptr(rstd)
    a.M, a.C, a.ldx, a.ldg, a.ldy = M, Cn, ldx, ldg, _mat(dX, "dX", dev, out=True)
    if param_grads:
        a.accumulate = 0 if dgamma is None else 1
        if dgamma is None:
            dgamma, dbeta = torch.empty(Cn, dtype=torch.float32, device=dev), torch.empty(Cn, dtype=torch.float32, device=dev)
        a.part_cap = lib.spb_layernorm_bwd_floats(M, Cn)
        part = torch.empty(a.part_cap, dtype=torch.float32, device=dev)
        a.part, a.dgamma, a.dbeta = _ptr(part), _ptr(dgamma), _ptr(dbeta)
    _call(dev, lib.spb_layernorm_bwd, "spb_layernorm_bwd", dtype_code(X, True), C.byref(a))
    return dX, dgamma, dbeta


class Packed8:
    """A matrix in e4m3 codes with one power-of-two scale for each block of 128 (include/spb_hip.h "8-bit packing"): codes uint8 [rows, K rounded up to
    128], scales uint8 (exponent + 127); block_rows 1 (quant8) or 128 (quant8_weight)."""
    __slots__ = ("codes", "scales", "K", "block_rows")

    def __init__(self, codes, scales, K, block_rows):
        self.codes, self.scales, self.K, self.block_rows = codes, scales, K, block_rows

    @staticmethod
    def empty(rows, K, block_rows, device):
        kb = (K + 127) // 128
        return Packed8(torch.empty(rows, kb * 128, dtype=torch.uint8, device=device),
                       torch.empty((rows + block_rows - 1) // block_rows, (kb + 3) // 4 * 4, dtype=torch.uint8, device=device), K, block_rows)

    @property
    def shape(self):
        return (self.codes.shape[0], self.K)


def _packed(P, name, dev, block_rows=None):
    if not isinstance(P, Packed8):
        raise RuntimeError("%s must be a Packed8 (quant8 / quant8_weight), got %s" % (name, type(P).__name__))
    if block_rows is not None and P.block_rows != block_rows:
        raise RuntimeError("%s must be packed in blocks of %d x 128" % (name, block_rows))
    rows, kb = P.codes.shape[0], (P.K + 127) // 128
    for t, shape in ((P.codes, (rows, kb * 128)), (P.scales, ((rows + P.block_rows - 1) // P.block_rows, (kb + 3) // 4 * 4))):
        if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous():
            raise RuntimeError("%s: codes and scales do not fit a packed [%d, %d] matrix" % (name, rows, P.K))
        if not t.is_cuda or (dev is not None and t.device != dev):
            raise RuntimeError("%s is on %s, expected %s" % (name, t.device, dev or "a GPU"))


def quant8(X):
    """X [M, K] packed in blocks of 1 x 128: operand of gemm8 and checkpoint for gemm8_wgrad"""
    ldx = _mat(X, "X")
    M, K = X.shape
    P = Packed8.empty(M, K, 1, X.device)
    _call(X.device, lib_of(X).spb_pack8_rows, "spb_pack8_rows", dtype_code(X, True), _ptr(X), ldx, M, K, _ptr(P.codes), _ptr(P.scales))
    return P


def quant8_weight(W, transpose=True):
    """W [N, K] packed in blocks of 128 x 128: (operand of Y = X W^T, packed transpose for dX = G W or None)"""
    ldw = _mat(W, "W")
    N, K = W.shape
    P = Packed8.empty(N, K, 128, W.device)
    T = Packed8.empty(K, N, 128, W.device) if transpose else None
    _call(W.device, lib_of(W).spb_pack8_weight, "spb_pack8_weight", dtype_code(W, True), _ptr(W), ldw, N, K, _ptr(P.codes), _ptr(P.scales),
          _ptr(T.codes) if transpose else None, _ptr(T.scales) if transpose else None)
    return P, T


def dequant8(P, dtype=torch.bfloat16, Y=None):
    """the values of a Packed8 (exact in bfloat16 and float32)"""
    _packed(P, "P", None)
    dev = P.codes.device
    if Y is None:
        Y = torch.empty(P.shape, dtype=dtype, device=dev)
    else:
        _like(Y, P.shape, dtype, "Y", dev)
    ldy = _mat(Y, "Y", dev, out=True)
    _call(dev, lib_of(Y).spb_unpack8, "spb_unpack8", dtype_code(Y, True), _ptr(P.codes), _ptr(P.scales), P.block_rows, P.shape[0], P.K, _ptr(Y), ldy)
    return Y


def gemm8(A, B, bias=None, dtype=torch.bfloat16, Y=None):
    """Y [M, N] = A [M, K] (quant8) times the transpose of B [N, K] (quant8_weight or quant8) + bias (float32 [N]).  dtype float32: the products run
    through the bfloat16 matrix instructions, where they are exact; 16-bit types: through the 8-bit ones."""
    _packed(A, "A", None, 1)
    dev = A.codes.device
    _packed(B, "B", dev)
    if A.K != B.K:
        raise RuntimeError("gemm8: A has %d columns, B has %d" % (A.K, B.K))
    M, N = A.shape[0], B.shape[0]
    _vec(bias, N, "bias", dev)
    if Y is None:
        Y = torch.empty(M, N, dtype=dtype, device=dev)
    else:
        _like(Y, (M, N), dtype, "Y", dev)
    a = A8.Gemm8Args()
    a.ldy = _mat(Y, "Y", dev, out=True)
    a.A, a.As, a.B, a.Bs, a.bias, a.Y = _ptr(A.codes), _ptr(A.scales), _ptr(B.codes), _ptr(B.scales), _ptr(bias), _ptr(Y)
    a.M, a.N, a.K, a.b_block_rows = M, N, A.K, B.block_rows
    lib, code = lib_of(Y), dtype_code(Y, True)
    a.ws_bytes = lib.spb_gemm8_bytes(code, M, N, A.K)
    if a.ws_bytes > 0:
        ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=dev)
        a.ws = _ptr(ws)
    _call(dev, lib.spb_gemm8, "spb_gemm8", code, C.byref(a))
    return Y


def gemm8_wgrad(G, X8, dW=None):
    """dW [N, K] (float32) = transpose of G [M, N] times the checkpoint X8 (quant8 of the layer's input [M, K]); dW given: accumulated into"""
    ldg = _mat(G, "G")
    dev = G.device
    _packed(X8, "X8", dev, 1)
    (M, N), K = G.shape, X8.K
    if X8.shape[0] != M:
        raise RuntimeError("gemm8_wgrad: G has %d rows, X8 has %d" % (M, X8.shape[0]))
    a = A8.Wgrad8Args()
    a.accumulate = 0 if dW is None else 1
    if dW is None:
        dW = torch.empty(N, K, dtype=torch.float32, device=dev)
    else:
        _like(dW, (N, K), torch.float32, "dW", dev)
    a.ldw = _mat(dW, "dW", dev, out=True)
    a.G, a.X, a.Xs, a.dW = _ptr(G), _ptr(X8.codes), _ptr(X8.scales), _ptr(dW)
    a.M, a.N, a.K, a.ldg = M, N, K, ldg
    lib, code = lib_of(G), dtype_code(G, True)
    a.ws_bytes = lib.spb_gemm8_wgrad_bytes(code, M, N, K)
    if a.ws_bytes > 0:
        ws = torch.empty(a.ws_bytes, dtype=torch.uint8, device=dev)
        a.ws = _ptr(ws)
    _call(dev, lib.spb_gemm8_wgrad, "spb_gemm8_wgrad", code, C.byref(a))
    return dW


def _act8(act):
    if act not in (L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU):
        raise RuntimeError("act8 knows ACT_GELU, ACT_GELU_TANH and ACT_SILU, got %r" % (act,))


def act8_fwd(X, act, Y=None):
    """(Y, P): Y = act(X) and P = X in 8 bits, the checkpoint act8_bwd reads.  Y: optional output of X's type, may be X itself."""
    _act8(act)
    ldx = _mat(X, "X")
    dev, (M, K) = X.device, X.shape
    if Y is None:
        Y = torch.empty(M, K, dtype=X.dtype, device=dev)
    else:
        _like(Y, X.shape, X.dtype, "Y", dev)
    P = Packed8.empty(M, K, 1, dev)
    _call(dev, lib_of(X).spb_act8_fwd, "spb_act8_fwd", dtype_code(X, True), act, _ptr(X), ldx, _ptr(Y), _mat(Y, "Y", dev, out=True), M, K,
          _ptr(P.codes), _ptr(P.scales))
    return Y, P


def act8_bwd(G, P, act, dX=None):
    """dX = G * act'(value of the checkpoint P).  dX: optional output of G's type, may be G itself."""
    _act8(act)
    ldg = _mat(G, "G")
    dev, (M, K) = G.device, G.shape
    _packed(P, "P", dev, 1)
    if P.shape != (M, K):
        raise RuntimeError("act8_bwd: G is %s, the checkpoint %s" % ((M, K), P.shape))
    if dX is None:
        dX = torch.empty(M, K, dtype=G.dtype, device=dev)
    else:
        _like(dX, G.shape, G.dtype, "dX", dev)
    _call(dev, lib_of(G).spb_act8_bwd, "spb_act8_bwd", dtype_code(G, True), act, _ptr(G), ldg, _ptr(P.codes), _ptr(P.scales), _ptr(dX),
          _mat(dX, "dX", dev, out=True), M, K)
    return dX


def debug_trread(inp, out):
    _need_cuda(inp, out)
    L.check(L.lib().spb_debug_trread(_ptr(inp), _ptr(out), _stream()), "spb_debug_trread")


class StreamFork:
    """`fork(to)`: everything enqueued on stream `to` afterwards runs behind everything the current stream holds now -- what
    `to.wait_stream(torch.cuda.current_stream())` does, without the event record that costs the CURRENT stream 6-9 us on this device
    (spb_fork_streams in include/spb_hip.h: a one-wave store kernel here, a one-wave gate kernel there; events inside a stream capture, with
    SPB_EVENT_FORKS=1 and under rocprofv3 counter collection).  One native object per source stream (serial numbers must be stored in
    order); joins -- the current stream waiting for `to` -- stay `wait_stream`: the waiting stream has to stall there anyway."""

    def __init__(self):
        self._h = {}

    def __call__(self, to, src=None):
        src = torch.cuda.current_stream(to.device) if src is None else src
        if src.cuda_stream == to.cuda_stream:
            return
        h = self._h.get(src.cuda_stream)
        if h is None:
            h = C.c_void_p()
            with torch.cuda.device(to.device):
                L.check(L.lib().spb_fork_create(C.byref(h)), "spb_fork_create")
            self._h[src.cuda_stream] = h
        L.check(L.lib().spb_fork_streams(h, C.c_void_p(src.cuda_stream), C.c_void_p(to.cuda_stream)), "spb_fork_streams")

    def __del__(self):
        try:
            for h in self._h.values():
                L.lib().spb_fork_destroy(h)
        except Exception:
            pass

    def __deepcopy__(self, memo):     # native handles are not copied: a copied module forks through objects of its own
        return StreamFork()

    def __reduce__(self):
        return (StreamFork, ())
