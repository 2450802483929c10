"""Thin torch-tensor front end of the per-kernel C-ABI entry points (used by the parity tests and by callers that
want a single fused op).  Tensors are device memory only; all arithmetic happens in libspb_hip.so.
"""
import ctypes as C
import os

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
# A call on a few rows is bound by this file, not by its kernel (12-22 us with the helpers above; like this quant8 and gemm8 take 7 us, layernorm_bwd with
# its five tensors and two launches 16 us): devices are compared as indices, argument structs are filled by position, and addresses are plain integers.

_TUNED = bool(os.environ.get("SPB_DEBUG") or os.environ.get("SPB_TUNING_LIB"))


def _lib8(dtype):
    if dtype is torch.float16:
        return L._lib_f16 or L.lib_f16()
    return L._lib if L._lib is not None and not _TUNED and L._tuning_depth == 0 else L.lib()


def _call(dev, fn, what, *args):
    if dev == torch._C._cuda_getDevice():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(dev))     # current_stream(dev).cuda_stream without the 3 us of its object
        if code:
            L.check(code, what)
    else:
        with torch.cuda.device(dev):
            L.check(fn(*args, torch.cuda.current_stream().cuda_stream), what)


def _mat(t, name, dev=None):
    """2-D operand: device memory, contiguous columns, one of the three types.  Returns (device, rows, columns, row stride, type code)."""
    code, d = _DT.get(t.dtype), t.get_device()
    if code is None:
        raise RuntimeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if d < 0:
        raise RuntimeError("speedplusbaseline_amd ops run on the GPU only (got a %s tensor for %s)" % (t.device, name))
    if dev is not None and d != dev:
        raise RuntimeError("%s is on device %d, the other operands on %d" % (name, d, dev))
    if t.dim() != 2:
        raise RuntimeError("%s must be 2-D, got shape %s" % (name, tuple(t.shape)))
    (rows, cols), (ld, one) = t.shape, t.stride()
    if one != 1 and cols > 1:
        raise RuntimeError("the columns of %s must be contiguous, got strides %s" % (name, t.stride()))
    return d, rows, cols, ld if rows > 1 else cols, code


def _like(t, shape, dtype, name, dev):
    """an operand or output of a known shape and type; returns its row stride"""
    if t.get_device() != dev or t.dtype != dtype or tuple(t.shape) != shape:
        raise RuntimeError("%s must be %s %s on device %s, got %s %s on %s" % (name, dtype, shape, dev, t.dtype, tuple(t.shape), t.device))
    return _mat(t, name)[3]


def _out(t, shape, dtype, name, dev):
    ld = _like(t, shape, dtype, name, dev)
    if ld < shape[1]:
        raise RuntimeError("the rows of %s overlap" % name)
    return ld


def _vec(t, n, name, dev):
    """address of a contiguous float32 vector of n elements, or None"""
    if t is None:
        return None
    if t.get_device() != dev or t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise RuntimeError("%s must be a contiguous float32 [%d] on device %s, got %s %s on %s" % (name, n, dev, t.dtype, tuple(t.shape), t.device))
    return t.data_ptr()


def layernorm_fwd(X, gamma=None, beta=None, eps=1e-5, Y=None):
    """Layer norm over the columns of X [M, C]: returns (Y, mean, rstd); mean and rstd (float32 [M]) are what layernorm_bwd needs.  gamma / beta:
    float32 [C] or None (1 / 0).  Y: optional output of X's type, may be X itself."""
    dev, M, Cn, ldx, code = _mat(X, "X")
    if Cn < 1:
        raise RuntimeError("layernorm needs at least one column")
    if Y is None:
        Y, ldy = X.new_empty((M, Cn)), Cn
    else:
        ldy = _out(Y, (M, Cn), X.dtype, "Y", dev)
    mean, rstd = torch.empty((2, M), dtype=torch.float32, device=X.device).unbind(0)
    a = A8.LayerNormArgs(X.data_ptr(), None, _vec(gamma, Cn, "gamma", dev), _vec(beta, Cn, "beta", dev), Y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                         None, None, None, 0, M, ldx, 0, ldy, Cn, eps, 0)
    _call(dev, _lib8(X.dtype).spb_layernorm_fwd, "spb_layernorm_fwd", code, C.byref(a))
    return Y, mean, rstd


def layernorm_bwd(G, X, mean, rstd, gamma=None, dgamma=None, dbeta=None, dX=None, param_grads=True):
    """Backward of layernorm_fwd: returns (dX, dgamma, dbeta).  dgamma / dbeta given: accumulated into (both or neither), otherwise new;
    param_grads=False: not computed (None).  dX: optional output, may be G itself."""
    dev, M, Cn, ldx, code = _mat(X, "X")
    ldg = _like(G, (M, Cn), X.dtype, "G", dev)
    if Cn < 1:
        raise RuntimeError("layernorm needs at least one column")
    if (dgamma is None) != (dbeta is None) or (dgamma is not None and not param_grads):
        raise RuntimeError("dgamma and dbeta are accumulated into together")
    if mean is None or rstd is None:
        raise RuntimeError("layernorm_bwd needs the forward's mean and rstd")
    if dX is None:
        dX, ldd = X.new_empty((M, Cn)), Cn
    else:
        ldd = _out(dX, (M, Cn), X.dtype, "dX", dev)
    lib = _lib8(X.dtype)
    cap, part, accumulate, dgp, dbp = 0, None, 0, None, None
    if param_grads:
        if dgamma is None:
            dgamma, dbeta = torch.empty((2, Cn), dtype=torch.float32, device=X.device).unbind(0)
            dgp, dbp = dgamma.data_ptr(), dbeta.data_ptr()
        else:
            accumulate, dgp, dbp = 1, _vec(dgamma, Cn, "dgamma", dev), _vec(dbeta, Cn, "dbeta", dev)
        cap = lib.spb_layernorm_bwd_floats(M, Cn)
        part = torch.empty(cap, dtype=torch.float32, device=X.device)
    a = A8.LayerNormArgs(X.data_ptr(), G.data_ptr(), _vec(gamma, Cn, "gamma", dev), None, dX.data_ptr(), _vec(mean, M, "mean", dev),
                         _vec(rstd, M, "rstd", dev), dgp, dbp, None if part is None else part.data_ptr(), cap, M, ldx, ldg, ldd, Cn, 0.0, accumulate)
    _call(dev, lib.spb_layernorm_bwd, "spb_layernorm_bwd", code, C.byref(a))
    return dX, dgamma, dbeta


class Packed8:
    """A matrix in e4m3 codes with one power-of-two scale for each block of 128 (include/spb_hip.h "8-bit packing"): codes uint8 [rows, K rounded up to
    128], scales uint8 (exponent + 127); block_rows 1 (quant8) or 128 (quant8_weight).
    A matrix made by `empty` owns one buffer, which nobody else can move, and keeps its device and addresses (1 us of a call's 7); copies (copy, pickle, torch.save) are
    built anew from the copied tensors.  One made of a caller's tensors asks them at every call."""
    __slots__ = ("K", "block_rows", "shape", "_rows", "_own", "_dev", "_qp", "_sp")

    def __init__(self, codes, scales, K, block_rows):
        if block_rows not in (1, 128) or K < 0 or codes.dim() != 2:
            raise RuntimeError("Packed8: block_rows must be 1 or 128 and the codes a matrix")
        rows = codes.shape[0]
        self.K, self.block_rows, self.shape, self._rows = K, block_rows, (rows, K), rows
        self._own, self._dev = (codes, scales), None
        self._check()

    def _check(self):
        """a caller's tensors: also at every call, since they may have been given other storage"""
        codes, scales = self._own
        kb, rows = (self.K + 127) // 128, self._rows
        for t, shape in ((codes, (rows, kb * 128)), (scales, ((rows + self.block_rows - 1) // self.block_rows, (kb + 3) // 4 * 4))):
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != codes.device:
                raise RuntimeError("Packed8: codes and scales do not fit a packed [%d, %d] matrix" % (rows, self.K))

    @staticmethod
    def empty(rows, K, block_rows, device):
        """uninitialised; codes and scales share one allocation"""
        kb = (K + 127) // 128
        buf = torch.empty(rows * kb * 128 + (rows + block_rows - 1) // block_rows * ((kb + 3) // 4 * 4), dtype=torch.uint8, device=device)
        return Packed8._around(buf, rows, K, block_rows)

    @staticmethod
    def _around(buf, rows, K, block_rows):
        self = Packed8.__new__(Packed8)
        self.K, self.block_rows, self.shape, self._rows = K, block_rows, (rows, K), rows
        self._own, self._dev, self._qp = buf, buf.get_device(), buf.data_ptr()
        self._sp = self._qp + rows * ((K + 127) // 128) * 128
        return self

    def __reduce__(self):
        if self._dev is None:
            return Packed8, (*self._own, self.K, self.block_rows)
        return Packed8._around, (self._own, self._rows, self.K, self.block_rows)

    @property
    def device(self):
        return (self._own[0] if self._dev is None else self._own).device

    @property
    def codes(self):
        if self._dev is None:
            return self._own[0]
        kp = (self.K + 127) // 128 * 128
        return self._own[:self._rows * kp].view(self._rows, kp)

    @property
    def scales(self):
        if self._dev is None:
            return self._own[1]
        kb = (self.K + 127) // 128
        return self._own[self._rows * kb * 128:].view((self._rows + self.block_rows - 1) // self.block_rows, (kb + 3) // 4 * 4)

    def _at(self):
        """addresses of the codes and the scales"""
        if self._dev is None:
            return self._own[0].data_ptr(), self._own[1].data_ptr()
        return self._qp, self._sp


def _packed(P, name, dev=None, block_rows=None):
    """checks a Packed8 operand; returns its device and the addresses of its codes and scales"""
    if not isinstance(P, Packed8):
        raise RuntimeError("%s must be a Packed8 (quant8 / quant8_weight), got %s" % (name, type(P).__name__))
    if block_rows is not None and P.block_rows != block_rows:
        raise RuntimeError("%s must be packed in blocks of %d x 128" % (name, block_rows))
    on = P._dev
    if on is None:
        P._check()
        on = P._own[0].get_device()
    if on < 0 or (dev is not None and on != dev):
        raise RuntimeError("%s is on %s, expected %s" % (name, P.device, "a GPU" if dev is None else "device %d" % dev))
    if P._dev is None:
        return on, *P._at()
    return on, P._qp, P._sp


def quant8(X):
    """X [M, K] packed in blocks of 1 x 128: operand of gemm8 and checkpoint for gemm8_wgrad"""
    dev, M, K, ldx, code = _mat(X, "X")
    P = Packed8.empty(M, K, 1, X.device)
    _call(dev, _lib8(X.dtype).spb_pack8_rows, "spb_pack8_rows", code, X.data_ptr(), ldx, M, K, P._qp, P._sp)
    return P


def quant8_weight(W, transpose=True):
    """W [N, K] packed in blocks of 128 x 128: (operand of Y = X W^T, packed transpose for dX = G W or None)"""
    dev, N, K, ldw, code = _mat(W, "W")
    P = Packed8.empty(N, K, 128, W.device)
    T = Packed8.empty(K, N, 128, W.device) if transpose else None
    _call(dev, _lib8(W.dtype).spb_pack8_weight, "spb_pack8_weight", code, W.data_ptr(), ldw, N, K, P._qp, P._sp,
          T._qp if transpose else None, T._sp if transpose else None)
    return P, T


def dequant8(P, dtype=torch.bfloat16, Y=None):
    """the values of a Packed8 (exact in bfloat16 and float32)"""
    dev, qp, sp = _packed(P, "P")
    if Y is None:
        Y = torch.empty(P.shape, dtype=dtype, device=P.device)
    ldy = _out(Y, P.shape, dtype, "Y", dev)
    _call(dev, _lib8(dtype).spb_unpack8, "spb_unpack8", _DT[dtype], qp, sp, P.block_rows, P._rows, P.K, Y.data_ptr(), ldy)
    return Y


def gemm8(A, B, bias=None, dtype=torch.bfloat16, Y=None):
    """Y [M, N] = A [M, K] (quant8) times the transpose of B [N, K] (quant8_weight or quant8) + bias (float32 [N]).  dtype float32, or up to
    16 rows: the products run through the bfloat16 matrix instructions, where they are exact; otherwise through the 8-bit ones."""
    dev, aq, a_s = _packed(A, "A", None, 1)
    _, bq, bs = _packed(B, "B", dev)
    if A.K != B.K:
        raise RuntimeError("gemm8: A has %d columns, B has %d" % (A.K, B.K))
    M, N, K = A._rows, B._rows, A.K
    if dtype not in _DT:
        raise RuntimeError("gemm8 writes float32, bfloat16 or float16, not %s" % dtype)
    if Y is None:
        Y, ldy = torch.empty((M, N), dtype=dtype, device=A.device), N
    else:
        ldy = _out(Y, (M, N), dtype, "Y", dev)
    lib, code = _lib8(dtype), _DT[dtype]
    need = lib.spb_gemm8_bytes(code, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=A.device) if need > 0 else None
    a = A8.Gemm8Args(aq, a_s, bq, bs, _vec(bias, N, "bias", dev), Y.data_ptr(),
                     None if ws is None else ws.data_ptr(), need, M, ldy, N, K, B.block_rows)
    _call(dev, lib.spb_gemm8, "spb_gemm8", code, C.byref(a))
    return Y


def gemm8_wgrad(G, X8, dW=None):
    """dW [N, K] (float32) = transpose of G [M, N] times the checkpoint X8 (quant8 of the layer's input [M, K]); dW given: accumulated into"""
    dev, M, N, ldg, code = _mat(G, "G")
    _, xq, xs = _packed(X8, "X8", dev, 1)
    K = X8.K
    if X8._rows != M:
        raise RuntimeError("gemm8_wgrad: G has %d rows, X8 has %d" % (M, X8._rows))
    accumulate = 0 if dW is None else 1
    if dW is None:
        dW, ldw = torch.empty((N, K), dtype=torch.float32, device=G.device), K
    else:
        ldw = _out(dW, (N, K), torch.float32, "dW", dev)
    lib = _lib8(G.dtype)
    need = lib.spb_gemm8_wgrad_bytes(code, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=G.device) if need > 0 else None
    a = A8.Wgrad8Args(G.data_ptr(), xq, xs, dW.data_ptr(), None if ws is None else ws.data_ptr(), need, M, ldg, ldw,
                      N, K, accumulate)
    _call(dev, lib.spb_gemm8_wgrad, "spb_gemm8_wgrad", code, C.byref(a))
    return dW


def _act8(act):
    if act not in (L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU):
        raise RuntimeError("act8 knows ACT_GELU, ACT_GELU_TANH and ACT_SILU, got %r" % (act,))


def act8_fwd(X, act, Y=None):
    """(Y, P): Y = act(X) and P = X in 8 bits, the checkpoint act8_bwd reads.  Y: optional output of X's type, may be X itself."""
    _act8(act)
    dev, M, K, ldx, code = _mat(X, "X")
    if Y is None:
        Y, ldy = X.new_empty((M, K)), K
    else:
        ldy = _out(Y, (M, K), X.dtype, "Y", dev)
    P = Packed8.empty(M, K, 1, X.device)
    _call(dev, _lib8(X.dtype).spb_act8_fwd, "spb_act8_fwd", code, act, X.data_ptr(), ldx, Y.data_ptr(), ldy, M, K, P._qp, P._sp)
    return Y, P


def act8_bwd(G, P, act, dX=None):
    """dX = G * act'(value of the checkpoint P).  dX: optional output of G's type, may be G itself."""
    _act8(act)
    dev, M, K, ldg, code = _mat(G, "G")
    _, qp, sp = _packed(P, "P", dev, 1)
    if P._rows != M or P.K != K:
        raise RuntimeError("act8_bwd: G is %s, the checkpoint %s" % ((M, K), P.shape))
    if dX is None:
        dX, ldd = G.new_empty((M, K)), K
    else:
        ldd = _out(dX, (M, K), G.dtype, "dX", dev)
    _call(dev, _lib8(G.dtype).spb_act8_bwd, "spb_act8_bwd", code, act, G.data_ptr(), ldg, qp, sp, dX.data_ptr(), ldd, M, K)
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
