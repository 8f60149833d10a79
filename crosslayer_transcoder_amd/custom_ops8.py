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
from .ops8 import Block8, gemm8

_DEV = "cuda"
_E4M3 = ops8.FORMATS["e4m3"]


def _u8(like: Tensor, *shape):
    return torch.empty(shape, dtype=torch.uint8, device=like.device)


def _form_shapes(L, rows, cols):
    up = ops8._up
    return (L, rows, up(cols)), (L, up(cols) // 128, up(rows))


# ---- one linear map per layer: the encoder (W [L, N, K] in memory) and the per-layer decoder (W [L, K, N]) -----------------
def _forward(x, W, b, kn, keep_x, keep_w):
    """-> y [T, L, N], kept x (codes, scale bytes), kept W (codes, scale bytes); None where not kept."""
    T, L, K = x.shape
    N = W.shape[2] if kn else W.shape[1]
    q, s, xt, xs, _ = ops8.pack8_raw(ops8._dense(x).transpose(0, 1), _E4M3, True, keep_x)
    # the contraction over K reads the [N, K] form, the input gradient the [K, N] form
    d, ds, t, ts, _ = ops8.pack8_raw(ops8._dense(W), _E4M3, keep_w or not kn, keep_w or kn, tiles=True)
    (f, fs), (g, gs) = ((t, ts), (d, ds)) if kn else ((d, ds), (t, ts))
    y = torch.empty((T, L, N), dtype=x.dtype, device=x.device)
    gemm8(Block8(q, s, T, K), Block8(f, fs, N, K), b, out=y.transpose(0, 1))
    return y, xt, xs, (g if keep_w else None), (gs if keep_w else None)


def _gradients(dy, xt, xs, w, ws, K, kn, need_dx, w_dtype, need_db):
    """-> dx [T, L, K], dW (shape of W), db fp32 [L, N]; None where not asked for (w_dtype None: no dW)."""
    T, L, N = dy.shape
    need_dw = w_dtype is not None
    # (the bias gradient rides along with a pack; alone it still takes one)
    q, s, qt, st, db = ops8.pack8_raw(ops8._dense(dy).transpose(0, 1), _E4M3, need_dx or not need_dw, need_dw, sums=need_db)
    dx = dW = None
    if need_dx:
        dx = torch.empty((T, L, K), dtype=dy.dtype, device=dy.device)
        gemm8(Block8(q, s, T, N), Block8(w, ws, K, N), out=dx.transpose(0, 1))
    if need_dw:
        xk, gk = Block8(xt, xs, K, T), Block8(qt, st, N, T)
        dW = gemm8(xk, gk, out_dtype=w_dtype) if kn else gemm8(gk, xk, out_dtype=w_dtype)
    return dx, dW, db


@torch.library.custom_op("clt_hip::linear8", mutates_args=(), device_types=_DEV)
def linear8(x: Tensor, W: Tensor, b: Optional[Tensor], kn: bool, keep_x: bool, keep_w: bool) -> List[Tensor]:
    """x [T, L, K], W [L, N, K] (kn: [L, K, N]) -> [y [T, L, N], kept x (codes, scale bytes), kept W (codes, scale bytes)];
    the kept tensors are empty where keep_x / keep_w is false."""
    return [_u8(x, 0) if t is None else t for t in _forward(x, W, b, kn, keep_x, keep_w)]


@linear8.register_fake
def _(x, W, b, kn, keep_x, keep_w):
    T, L, K = x.shape
    N = W.shape[2] if kn else W.shape[1]
    (xd, xs), (wd, ws) = _form_shapes(L, K, T), _form_shapes(L, K, N)
    e = (0,)
    return [x.new_empty(T, L, N)] + [_u8(x, *sh) for sh in (xd if keep_x else e, xs if keep_x else e, wd if keep_w else e, ws if keep_w else e)]


@torch.library.custom_op("clt_hip::linear8_bwd", mutates_args=(), device_types=_DEV)
def linear8_bwd(dy: Tensor, xt: Tensor, xs: Tensor, w: Tensor, ws: Tensor, K: int, kn: bool, need_dx: bool, w_dtype: Optional[torch.dtype],
                need_db: bool) -> List[Tensor]:
    """-> [dx [T, L, K], dW (shape of W), db fp32 [L, N]], empty where not asked for (w_dtype None: no dW)."""
    return [dy.new_empty(0) if t is None else t for t in _gradients(dy, xt, xs, w, ws, K, kn, need_dx, w_dtype, need_db)]


@linear8_bwd.register_fake
def _(dy, xt, xs, w, ws, K, kn, need_dx, w_dtype, need_db):
    T, L, N = dy.shape
    dW = dy.new_empty(0) if w_dtype is None else dy.new_empty((L, K, N) if kn else (L, N, K), dtype=w_dtype)
    return [dy.new_empty(T, L, K) if need_dx else dy.new_empty(0), dW, dy.new_empty((L, N), dtype=torch.float32) if need_db else dy.new_empty(0)]


def _setup(ctx, inputs, output):
    x, W, b, ctx.kn, ctx.keep_x, ctx.keep_w = inputs
    ctx.K, ctx.w_dtype, ctx.b_dtype = x.shape[2], W.dtype, None if b is None else b.dtype
    ctx.b_shape = None if b is None else b.shape
    ctx.save_for_backward(*output[1:])


def _backward(ctx, grads):
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    need_b = need_b and ctx.b_dtype is not None
    if (need_w and not ctx.keep_x) or (need_x and not ctx.keep_w):
        raise RuntimeError("linear8 was called without keeping what this gradient needs (keep_x for dW, keep_w for dx)")
    dx, dW, db = torch.ops.clt_hip.linear8_bwd(grads[0], *ctx.saved_tensors, ctx.K, ctx.kn, need_x, ctx.w_dtype if need_w else None, need_b)
    return dx if need_x else None, dW if need_w else None, db.to(ctx.b_dtype).reshape(ctx.b_shape) if need_b else None, None, None, None


linear8.register_autograd(_backward, setup_context=_setup)


class _Linear8(torch.autograd.Function):
    """The same two functions without the dispatcher's Python layers, for eager calls (a forward and backward of a few tokens:
    400 us of host time through the registered ops)."""

    @staticmethod
    def forward(ctx, x, W, b, kn):
        y, *kept = _forward(x, W, b, kn, ctx.needs_input_grad[1], ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        ctx.kn, ctx.K, ctx.w_dtype, ctx.b = kn, x.shape[2], W.dtype, None if b is None else (b.dtype, b.shape)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dW, db = _gradients(dy, *ctx.saved_tensors, ctx.K, ctx.kn, need_x, ctx.w_dtype if need_w else None, need_b)
        return dx, dW, db.to(ctx.b[0]).reshape(ctx.b[1]) if need_b else None, None


def _linear(x, W, b, kn):
    if x.dim() != 3 or W.dim() != 3 or W.shape[0] != x.shape[1] or W.shape[1 if kn else 2] != x.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} ([tokens, layers, features]) does not match W {tuple(W.shape)}")
    if torch.compiler.is_compiling():
        grad = torch.is_grad_enabled()
        return torch.ops.clt_hip.linear8(x, W, b, kn, grad and W.requires_grad, grad and x.requires_grad)[0]
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
