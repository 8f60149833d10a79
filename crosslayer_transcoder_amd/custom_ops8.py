"""Linear maps that contract in 8-bit block-scaled form and keep their input in 8 bits for the backward pass, as dispatcher ops
beside the fp32 / 16-bit ones of custom_ops.py (reference model/clt.py:157-165, 241-248, 334-343): `encoder8`, `plt_decoder8`,
`clt_decoder8` take the arguments of `clt_hip::encoder`, `plt_decoder`, `clt_decoder` and are differentiable in all of them.

Forward: y = X8 W8 + b, X8 the input with blocks of 128 along the contraction, W8 the weight in 128 x 128 tiles.  Kept for the
backward pass instead of the input (4 or 2 bytes an element): its transposed 8-bit copy with blocks of 128 tokens, written by
the same read (1 byte), and W8 in the orientation the input gradient contracts.  Backward, g8 / g8t the incoming gradient in
the same two forms: dx = g8 W8^T, dW = X8t g8t^T, db = the sum of g itself, taken by the pass that packs it.  These are the
straight-through gradients: rounding to 8 bits counts as the identity.

y and dx have x's type (dx of the cross-layer decoder is summed in fp32 first), dW has W's, db has b's."""
from typing import List, Optional

import torch
from torch import Tensor

from . import ops8
from ._lib import lib
from .ops8 import _DT, _call, _up

_DEV = "cuda"
_E4M3 = ops8.FORMATS["e4m3"]


# Bytes of the held forms.  The kept buffer is one allocation: x transposed (codes [L, K, up(T)], scale bytes [L, up(T) / 128, up(K)]),
# then W for the input gradient (codes [L, K, up(N)], scale bytes [L, up(N) / 128, up(K)]), either part only where it is kept.
def _held(L, rows, cols):
    c = _up(cols)
    return L * rows * c, L * (c // 128) * _up(rows)


def _kept_bytes(T, L, K, N, keep_x, keep_w):
    return (sum(_held(L, K, T)) if keep_x else 0) + (sum(_held(L, K, N)) if keep_w else 0)


def _forward(x, W, b, kn, keep_x, keep_w):
    """x [T, L, K], W [L, N, K] (kn: [L, K, N]) -> y [T, L, N], the kept buffer."""
    x, W = ops8._dense(x, (3,)), ops8._dense(W, (3,))
    T, L, K = x.shape
    N = W.shape[2] if kn else W.shape[1]
    dev = x.device
    if W.device != dev:
        raise ValueError("x and W are on different devices")
    if not (L and K and N):
        raise ValueError(f"empty map: x {tuple(x.shape)}, W {tuple(W.shape)}")
    b = ops8._bias(b, L, N, dev)
    y = torch.empty((T, L, N), dtype=x.dtype, device=dev)
    kept = torch.empty(_kept_bytes(T, L, K, N, keep_x, keep_w), dtype=torch.uint8, device=dev)
    if not T and not keep_w:
        return y, kept
    (nq, ns), (nf, nfs) = _held(L, T, K), _held(L, N, K)
    tmp = torch.empty(nq + ns + nf + nfs, dtype=torch.uint8, device=dev)
    q = tmp.data_ptr()
    s, f = q + nq, q + nq + ns
    fs = f + nf
    xt = wk = xs = ws = None
    at = kept.data_ptr()
    if keep_x:
        n, ns_ = _held(L, K, T)
        xt, xs = at, at + n
        at += n + ns_
    if keep_w:
        wk, ws = at, at + _held(L, K, N)[0]
    # the contraction over K reads the [N, K] form, the input gradient the [K, N] form
    d, ds, t, ts = (wk, ws, f, fs) if kn else (f, fs, wk, ws)
    with ops8._on(dev):
        st = ops8._stream(dev)
        R, C = W.shape[1:]
        _call(lib.clt_pack8, W.data_ptr(), _DT[W.dtype], W.stride(1), W.stride(0), L, R, C, _E4M3, 1, d, ds, t, ts, None, None, 0, st)
        if T:
            _call(lib.clt_pack8, x.data_ptr(), _DT[x.dtype], x.stride(0), x.stride(1), L, T, K, _E4M3, 0, q, s, xt, xs, None, None, 0, st)
            _gemm((q, s, L, T), (f, fs, L, N), K, y, L * N, N, b, N, st)
    return y, kept


def _gemm(a, b, K, out, ldc, cb, bias, nbias, st):
    """clt_gemm8 of densely held e4m3 operands (codes, scale bytes, batch, rows) contracting over K."""
    (aq, as_, L, M), (bq, bs, _, N) = a, b
    k = _up(K)
    sa, sb = _up(M), _up(N)
    nws = lib.clt_gemm8_workspace_bytes(M, N, K, L)
    ws = torch.empty(nws, dtype=torch.uint8, device=out.device) if nws else None
    _call(lib.clt_gemm8, aq, as_, _E4M3, k, sa, M * k, k // 128 * sa, bq, bs, _E4M3, k, sb, N * k, k // 128 * sb, out.data_ptr(),
          _DT[out.dtype], ldc, cb, bias.data_ptr() if bias is not None else None, nbias, M, N, K, L, 0,
          ws.data_ptr() if nws else None, nws, st)


def _gradients(dy, kept, K, kn, has_x, need_dx, w_dtype, need_db):
    """-> dx [T, L, K], dW (shape of W), db fp32 [L, N]; None where not asked for (w_dtype None: no dW).  has_x: x is in `kept`."""
    dy = ops8._dense(dy, (3,))
    T, L, N = dy.shape
    dev = dy.device
    need_dw = w_dtype is not None
    dx = torch.empty((T, L, K), dtype=dy.dtype, device=dev) if need_dx else None
    dW = torch.empty((L, K, N) if kn else (L, N, K), dtype=w_dtype, device=dev) if need_dw else None
    db = torch.empty((L, N), dtype=torch.float32, device=dev) if need_db else None
    if need_db and not T:
        db.zero_()
    (nq, ns), (nt, nts) = _held(L, T, N), _held(L, N, T)
    nws = lib.clt_pack8_sums_workspace_bytes(L, T, N) if need_db and T else 0
    along = need_dx or not need_dw                     # (the bias gradient rides along with a pack; alone it still takes one)
    tmp = torch.empty((nq + ns if along else 0) + (nt + nts if need_dw else 0) + nws, dtype=torch.uint8, device=dev)
    at = tmp.data_ptr()
    q = s = qt = qs = None
    if along:
        q, s = at, at + nq
        at += nq + ns
    if need_dw:
        qt, qs = at, at + nt
        at += nt + nts
    xt = kept.data_ptr()
    xs = xt + _held(L, K, T)[0]
    wk = xt + (sum(_held(L, K, T)) if has_x else 0)
    with ops8._on(dev):
        st = ops8._stream(dev)
        if T:
            _call(lib.clt_pack8, dy.data_ptr(), _DT[dy.dtype], dy.stride(0), dy.stride(1), L, T, N, _E4M3, 0, q, s, qt, qs,
                  db.data_ptr() if need_db else None, at if nws else None, nws, st)
            if need_dx:
                _gemm((q, s, L, T), (wk, wk + _held(L, K, N)[0], L, K), N, dx, L * K, K, None, 0, st)
        if need_dw:
            xk, gk = (xt, xs, L, K), (qt, qs, L, N)
            _gemm(*((xk, gk) if kn else (gk, xk)), T, dW, dW.shape[2], dW.shape[1] * dW.shape[2], None, 0, st)
    return dx, dW, db


@torch.library.custom_op("clt_hip::linear8", mutates_args=(), device_types=_DEV)
def linear8(x: Tensor, W: Tensor, b: Optional[Tensor], kn: bool, keep_x: bool, keep_w: bool) -> List[Tensor]:
    """x [T, L, K], W [L, N, K] (kn: [L, K, N]) -> [y [T, L, N], the bytes kept for the backward pass]: x where dW will be asked for
    (keep_x), W where dx will be (keep_w)."""
    return list(_forward(x, W, b, kn, keep_x, keep_w))


@linear8.register_fake
def _(x, W, b, kn, keep_x, keep_w):
    T, L, K = x.shape
    N = W.shape[2] if kn else W.shape[1]
    return [x.new_empty(T, L, N), x.new_empty(_kept_bytes(T, L, K, N, keep_x, keep_w), dtype=torch.uint8)]


@torch.library.custom_op("clt_hip::linear8_bwd", mutates_args=(), device_types=_DEV)
def linear8_bwd(dy: Tensor, kept: Tensor, K: int, kn: bool, has_x: bool, need_dx: bool, w_dtype: Optional[torch.dtype], need_db: bool) -> List[Tensor]:
    """-> [dx [T, L, K], dW (shape of W), db fp32 [L, N]], empty where not asked for (w_dtype None: no dW)."""
    return [dy.new_empty(0) if t is None else t for t in _gradients(dy, kept, K, kn, has_x, need_dx, w_dtype, need_db)]


@linear8_bwd.register_fake
def _(dy, kept, K, kn, has_x, need_dx, w_dtype, need_db):
    T, L, N = dy.shape
    dW = dy.new_empty(0) if w_dtype is None else dy.new_empty((L, K, N) if kn else (L, N, K), dtype=w_dtype)
    return [dy.new_empty(T, L, K) if need_dx else dy.new_empty(0), dW, dy.new_empty((L, N), dtype=torch.float32) if need_db else dy.new_empty(0)]


def _setup(ctx, inputs, output):
    x, W, b, ctx.kn, ctx.keep_x, ctx.keep_w = inputs
    ctx.K, ctx.w_dtype, ctx.b = x.shape[2], W.dtype, None if b is None else (b.dtype, b.shape)
    ctx.save_for_backward(output[1])


def _backward(ctx, grads):
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    if (need_w and not ctx.keep_x) or (need_x and not ctx.keep_w):
        raise RuntimeError("linear8 was called without keeping what this gradient needs (keep_x for dW, keep_w for dx)")
    dx, dW, db = torch.ops.clt_hip.linear8_bwd(grads[0], ctx.saved_tensors[0], ctx.K, ctx.kn, ctx.keep_x, need_x, ctx.w_dtype if need_w else None, need_b)
    return dx if need_x else None, dW if need_w else None, db.to(ctx.b[0]).reshape(ctx.b[1]) if need_b else None, None, None, None


linear8.register_autograd(_backward, setup_context=_setup)


class _Linear8(torch.autograd.Function):
    """The same two functions without the dispatcher's Python layers, for eager calls (a forward and backward of a few tokens:
    400 us of host time through the registered ops)."""

    @staticmethod
    def forward(ctx, x, W, b, kn):
        y, kept = _forward(x, W, b, kn, ctx.needs_input_grad[1], ctx.needs_input_grad[0])
        ctx.save_for_backward(kept)
        ctx.kn, ctx.K, ctx.has_x, ctx.w_dtype, ctx.b = kn, x.shape[2], ctx.needs_input_grad[1], W.dtype, None if b is None else (b.dtype, b.shape)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dW, db = _gradients(dy, ctx.saved_tensors[0], ctx.K, ctx.kn, ctx.has_x, need_x, ctx.w_dtype if need_w else None, need_b)
        if need_b and ctx.b != (torch.float32, db.shape):
            db = db.to(ctx.b[0]).reshape(ctx.b[1])
        return dx, dW, db, None


def _linear(x, W, b, kn):
    if x.dim() != 3 or W.dim() != 3 or W.shape[0] != x.shape[1] or W.shape[1 if kn else 2] != x.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} ([tokens, layers, features]) does not match W {tuple(W.shape)}")
    if torch.compiler.is_compiling():
        grad = torch.is_grad_enabled()
        return torch.ops.clt_hip.linear8(x, W, b, kn, grad and W.requires_grad, grad and x.requires_grad)[0]
    if not torch.is_grad_enabled():
        return _forward(x, W, b, kn, False, False)[0]
    return _Linear8.apply(x, W, b, kn)


def encoder8(xs: Tensor, W: Tensor, b: Optional[Tensor]) -> Tensor:
    """pre [B, L, F] = xs [B, L, d] @ W [L, d, F] + b [L, F] in 8-bit block-scaled form (`clt_hip::encoder`'s arguments).  W in its
    feature-major storage or dense: either is packed as it lies."""
    if W.dim() == 3 and not W.is_contiguous() and W.permute(0, 2, 1).is_contiguous():
        return _linear(xs, W.permute(0, 2, 1), b, False)
    return _linear(xs, W, b, True)


def plt_decoder8(feat: Tensor, W: Tensor, b: Optional[Tensor]) -> Tensor:
    """recons [B, L, d] = feat [B, L, F] @ W [L, F, d] + b [L, d] (`clt_hip::plt_decoder`'s arguments)."""
    return _linear(feat, W, b, True)


#: names of the registered ops, for tests and introspection
REGISTERED8 = ("linear8", "linear8_bwd")
