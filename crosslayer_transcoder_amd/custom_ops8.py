"""Linear maps that contract in 8-bit block-scaled form and keep their input in 8 bits for the backward pass, as dispatcher ops
beside the fp32 / 16-bit ones of custom_ops.py (reference model/clt.py:157-165, 241-248, 334-343): `encoder8`, `plt_decoder8`,
`clt_decoder8` take the arguments of `clt_hip::encoder`, `plt_decoder`, `clt_decoder` and are differentiable in all of them.

Forward: y = X8 W8 + b, X8 the input with blocks of 128 along the contraction, W8 the weight in 128 x 128 tiles.  Kept for the
backward pass instead of the input (4 or 2 bytes an element): its transposed 8-bit copy with blocks of 128 tokens, written by
the same read (1 byte), and W8 in the orientation the input gradient contracts.  Backward, g8 / g8t the incoming gradient in
the same two forms: dx = g8 W8^T, dW = X8t g8t^T, db = the sum of g itself, taken by the pass that packs it.  These are the
straight-through gradients: rounding to 8 bits counts as the identity.

y and dx have x's type, dW has W's, db has b's.  A product with a bf16 result uses the 8-bit matrix instructions, which align products
to about 14 bits (`ops8.gemm8`), one with an fp32 or fp16 result is exact up to fp32 sums: x in fp32 or fp16 asks for that.

A training step can be captured into a graph, forward and backward, as long as no eager graph of the same leaves is alive then (torch's
own rule: the engine would wait for the stream that graph was made on)."""
from typing import List, Optional

import torch
from torch import Tensor

from . import ops8
from ._lib import lib
from .ops8 import _DT, _call, _up

_DEV = "cuda"
_E4M3 = ops8.FORMATS["e4m3"]


def _kept_bytes(T, L, K, N, keep_x, keep_w):
    """clt_linear8_kept_bytes, of symbolic sizes too: codes and scale bytes of x [K, T] and of W [K, N]."""
    def held(rows, cols):
        return L * (rows * _up(cols) + _up(cols) // 128 * _up(rows))
    return (held(K, T) if keep_x else 0) + (held(K, N) if keep_w else 0)


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _check(x, W, kn):
    """Refuses what does not fit: the kernels take x's sizes for W's.  The op's body, its fake and the eager functions all come here
    (ops8._bias: the bias) -> T, L, K, N."""
    sx, sw = x.shape, W.shape
    if len(sx) != 3 or len(sw) != 3 or sw[0] != sx[1] or sw[1 if kn else 2] != sx[2]:
        raise ValueError(f"x {tuple(sx)} ([tokens, layers, features]) does not match W {tuple(sw)}")
    if W.device != x.device:
        raise ValueError("x and W are on different devices")
    return (*sx, sw[2 if kn else 1])


def _forward(x, W, b, kn, keep_x, keep_w):
    """x [T, L, K], W [L, N, K] (kn: [L, K, N]) -> y [T, L, N], the kept buffer."""
    T, L, K, N = _check(x, W, kn)
    b = ops8._bias(b, L, N, x.device)
    x, W = ops8._dense(x, (3,)), ops8._dense(W, (3,))
    dev = x.device
    if not (L and K and N):
        raise ValueError(f"empty map: x {tuple(x.shape)}, W {tuple(W.shape)}")
    y = torch.empty((T, L, N), dtype=x.dtype, device=dev)
    kept = _bytes(lib.clt_linear8_kept_bytes(T, L, K, N, keep_x, keep_w), dev)
    nws = lib.clt_linear8_forward_workspace_bytes(T, L, K, N)
    ws = _bytes(nws, dev)
    with ops8._on(dev):
        _call(lib.clt_linear8_forward, x.data_ptr(), _DT[x.dtype], x.stride(0), x.stride(1), W.data_ptr(), _DT[W.dtype], W.stride(1), W.stride(0), kn,
              b.data_ptr() if b is not None else None, y.data_ptr(), T, L, K, N, keep_x, keep_w, kept.data_ptr(), ws.data_ptr(), nws, ops8._stream(dev))
    return y, kept


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
    if need_dx or need_dw or need_db:
        nws = lib.clt_linear8_backward_workspace_bytes(T, L, K, N, need_dx, need_dw, need_db)
        ws = _bytes(nws, dev)
        with ops8._on(dev):
            _call(lib.clt_linear8_backward, dy.data_ptr(), _DT[dy.dtype], dy.stride(0), dy.stride(1), kept.data_ptr(), has_x, kn, T, L, K, N,
                  dx.data_ptr() if need_dx else None, dW.data_ptr() if need_dw else None, _DT[w_dtype] if need_dw else 0,
                  db.data_ptr() if need_db else None, ws.data_ptr(), nws, ops8._stream(dev))
    return dx, dW, db


@torch.library.custom_op("clt_hip::linear8", mutates_args=(), device_types=_DEV)
def linear8(x: Tensor, W: Tensor, b: Optional[Tensor], kn: bool, keep_x: bool, keep_w: bool) -> List[Tensor]:
    """x [T, L, K], W [L, N, K] (kn: [L, K, N]) -> [y [T, L, N], the bytes kept for the backward pass]: x where dW will be asked for
    (keep_x), W where dx will be (keep_w)."""
    return list(_forward(x, W, b, kn, keep_x, keep_w))


@linear8.register_fake
def _(x, W, b, kn, keep_x, keep_w):
    T, L, K, N = _check(x, W, kn)
    ops8._bias(b, L, N, x.device)
    return [x.new_empty(T, L, N), x.new_empty(_kept_bytes(T, L, K, N, keep_x, keep_w), dtype=torch.uint8)]


def _check_type(w_dtype):
    if w_dtype is not None and w_dtype not in _DT:
        raise TypeError(f"weight gradients are float32, bfloat16 or float16, got {w_dtype}")


@torch.library.custom_op("clt_hip::linear8_bwd", mutates_args=(), device_types=_DEV)
def linear8_bwd(dy: Tensor, kept: Tensor, K: int, kn: bool, has_x: bool, need_dx: bool, w_dtype: Optional[torch.dtype], need_db: bool) -> List[Tensor]:
    """-> [dx [T, L, K], dW (shape of W), db fp32 [L, N]], empty where not asked for (w_dtype None: no dW)."""
    T, L, N = dy.shape
    if kept.dtype != torch.uint8 or not kept.is_contiguous() or kept.device != dy.device or kept.numel() < _kept_bytes(T, L, K, N, has_x, need_dx):
        raise ValueError("`kept` is not what linear8 kept for this gradient")
    if w_dtype is not None and not has_x:
        raise ValueError("the weights' gradient needs the input that linear8 keeps with keep_x")
    _check_type(w_dtype)
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


_PLAIN = frozenset((Tensor, torch.nn.Parameter, type(None)))
_transforms = torch._C._functorch.peek_interpreter_stack


def _dispatched(*tensors):
    """Whether a call has to be the registered op: something compiles, traces, transforms or watches what runs (none of them would see a
    launch on an address), or a tensor is of a class with its own dispatch."""
    return (torch.compiler.is_compiling() or ops8._modes() > 0 or ops8._tracing() is not None or _transforms() is not None or
            not _PLAIN.issuperset(map(type, tensors)))


class _Linear8(torch.autograd.Function):
    """The same two functions without the dispatcher's Python layers, for eager calls that nothing watches (a forward and backward of
    a few tokens: 400 us of host time through the registered ops)."""

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
    if _dispatched(x, W, b):
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


# ---- cross-layer decoder: recons[:, l] = feat[:, :l+1].flatten(1) @ W_l.flatten(0, 1) + b[l] (reference model/clt.py:334-343) ----------
# Forward, blocks along the flattened (source layer, feature) axis: the features are packed once and target layer l contracts over the
# first (l + 1) F columns.  Gradient of source layer s: one product over the flattened (target layer, output) axis from s on,
#   dfeat[:, s] = [g_s .. g_{L-1}] [W_s[s]; ..; W_{L-1}[s]]^T,
# whose right operand the packing of each W_l fills in, block of columns by block of columns.  Both need borders between layers that are
# borders between blocks.  Where d is no multiple of 128 the L products of the targets are added up in fp32 instead (forward and
# backward of 12 layers, d = 768, 8192 features, 4096 tokens in fp32: 14.8 ms that way, 12.0 ms this way), and where F is none every prefix of the features is packed by itself.
def _clt_aligned(F, d):
    return F % ops8.BLOCK == 0 and d % ops8.BLOCK == 0


# The right operands of all source layers in [H, F, (L + 1) d], H = (L + 1) // 2: row p holds source layer p (targets p .. L - 1) and behind
# it source layer L - 1 - p (targets L - 1 - p .. L - 1), which fill it exactly (a middle layer's own row is half empty).
def _clt_source(s, L, d):
    """-> (row, first column) of source layer s."""
    return (s, 0) if s < (L + 1) // 2 else (L - 1 - s, (s + 1) * d)


def _clt_kept_shapes(B, L, F, d, keep_x, keep_w):
    """Shapes of the kept uint8 tensors: [x transposed (codes, scale bytes)] + [codes, scale bytes] of all source layers' operands, or of every
    W_l where the borders are not the blocks'."""
    def form(rows, cols):
        return [(1, rows, _up(cols)), (1, _up(cols) // 128, _up(rows))]
    shapes = form(L * F, B) if keep_x else []
    if keep_w and _clt_aligned(F, d):
        shapes += [((L + 1) // 2, F, (L + 1) * d), ((L + 1) // 2, (L + 1) * d // 128, F)]
    elif keep_w:
        for l in range(L):
            shapes += form((l + 1) * F, d)
    return shapes


def _clt_pack_weight(W, l, L, kq, ks, tq, ts, st):
    """W_l [l + 1, F, d] -> its transpose [d, (l + 1) F] (at tq, ts) and its columns of every source layer's operand (at kq, ks; or None)."""
    n, F, d = W.shape
    H, pitch, K = (L + 1) // 2, (L + 1) * d, (l + 1) * F
    for s0, s1 in ((0, min(n, H)), (H, n)):                  # (the layers of the second half lie the other way round)
        if s0 >= s1:
            continue
        p, c = _clt_source(s0, L, d)
        c += (l - s0) * d                                    # (one source layer further, this target lies d columns further left or right)
        step, left = (1, d) if s0 == 0 else (-1, 0)
        _call(lib.clt_pack8_into, W.data_ptr() + s0 * W.stride(0) * W.element_size(), _DT[W.dtype], W.stride(1), W.stride(0), s1 - s0, F, d, _E4M3, 1,
              kq + p * F * pitch + c if kq else None, ks + (p * pitch + c) // 128 * F if kq else None, pitch, step * F * pitch - left,
              (step * pitch - left) // 128 * F, tq + s0 * F, ts + s0 * F // 128 * d, K, F, F // 128 * d, None, None, 0, st)


def _product(a, b, K, c, dtype, ldc, bias, device, st):
    """One clt_gemm8 of operands (codes, scale bytes, their pitches, rows) into c, all addresses."""
    (aq, as_, lda, ldas, M), (bq, bs, ldb, ldbs, N) = a, b
    nws = lib.clt_gemm8_workspace_bytes(M, N, K, 1)
    ws = _bytes(nws, device) if nws else None
    _call(lib.clt_gemm8, aq, as_, _E4M3, lda, ldas, 0, 0, bq, bs, _E4M3, ldb, ldbs, 0, 0, c, dtype, ldc, 0, bias, 0, M, N, K, 1, 0,
          ws.data_ptr() if nws else None, nws, st)


def _clt_check(feat, b, Ws):
    """As _check: every W_l is addressed with its place in the features' layout."""
    if feat.dim() != 3 or not Ws or len(Ws) != feat.shape[1] or any(W.dim() != 3 or tuple(W.shape) != (l + 1, feat.shape[2], Ws[0].shape[2]) for l, W in enumerate(Ws)):
        raise ValueError(f"features {tuple(feat.shape)} do not match the decoder weights {[tuple(W.shape) for W in Ws]}")
    if any(W.device != feat.device or W.dtype != Ws[0].dtype for W in Ws):
        raise ValueError("the decoder weights are of one type, on the features' device")
    if b is not None and (tuple(b.shape) != (len(Ws), Ws[0].shape[2]) or b.device != feat.device):
        raise ValueError(f"bias {tuple(b.shape)} does not match {len(Ws)} layers of {Ws[0].shape[2]} on the features' device")


def _clt_forward(feat, b, Ws, keep_x, keep_w):
    """-> recons [B, L, d], the kept tensors."""
    _clt_check(feat, b, Ws)
    feat = ops8._dense(feat, (3,)).contiguous()
    B, L, F = feat.shape
    d = Ws[0].shape[2]
    if not (L and F and d):
        raise ValueError(f"empty map: features {tuple(feat.shape)}, W_0 {tuple(Ws[0].shape)}")
    dev = feat.device
    flat = feat.view(B, L * F)
    out = torch.empty((B, L, d), dtype=feat.dtype, device=dev)
    b = ops8._bias(b, L, d, dev)
    whole = F % ops8.BLOCK == 0
    q, s, xt, xs, _ = ops8.pack8_raw(flat.unsqueeze(0), _E4M3, whole, keep_x) if whole or keep_x else (None,) * 5
    kept = [xt, xs] if keep_x else []
    if _clt_aligned(F, d):
        k = [_bytes(shape, dev) for shape in _clt_kept_shapes(B, L, F, d, False, keep_w)]
        kq, ks = (t.data_ptr() for t in k) if keep_w else (None, None)
        tmp = _bytes(d * L * F + L * F // 128 * d, dev)      # one target layer's operand after the other
        tq, ts, es = tmp.data_ptr(), tmp.data_ptr() + d * L * F, out.element_size()
        with ops8._on(dev):
            st = ops8._stream(dev)
            for l, W in enumerate(Ws):
                K = (l + 1) * F
                _clt_pack_weight(ops8._dense(W, (3,)), l, L, kq, ks, tq, ts, st)
                if B:
                    _product((q.data_ptr(), s.data_ptr(), L * F, _up(B), B), (tq, ts, K, d, d), K, out.data_ptr() + l * d * es, _DT[out.dtype], L * d,
                             b.data_ptr() + 4 * l * d if b is not None else None, dev, st)
        return out, kept + k
    x = ops8.Block8(q, s, B, L * F) if whole else None
    for l, W in enumerate(Ws):
        K = (l + 1) * F
        dq, ds, tq, ts, _ = ops8.pack8_raw(ops8._dense(W, (3,)).reshape(1, K, d), _E4M3, keep_w, True, tiles=True)
        if keep_w:
            kept += [dq, ds]
        ops8.gemm8(x.first_columns(K) if whole else ops8.quantize8(flat[:, :K]), ops8.Block8(tq, ts, d, K), None if b is None else b[l:l + 1],
                   out=out[:, l].unsqueeze(0))
    return out, kept


def _clt_gradients(g, kept, F, has_x, need_dx, w_dtypes, need_db):
    """-> dfeat [B, L, F] of g's type, [dW_l [l + 1, F, d]], db fp32 [L, d]; None where not asked for (w_dtypes empty: no dW)."""
    g = ops8._dense(g, (3,))
    B, L, d = g.shape
    dev = g.device
    ws = kept[2:] if has_x else kept
    dx, dWs = None, None
    if _clt_aligned(F, d):
        # one matrix [B, L d]; its transpose holds layer l's in rows l d ..
        q, s, qt, qs, db = ops8.pack8_raw(g.reshape(1, B, L * d), _E4M3, need_dx or not w_dtypes, bool(w_dtypes), sums=need_db)
        t, pitch = _up(B), (L + 1) * d
        with ops8._on(dev):
            st = ops8._stream(dev)
            if need_dx:
                dx = torch.empty((B, L, F), dtype=g.dtype, device=dev)
                wq, wsc = ws[0].data_ptr(), ws[1].data_ptr()
                for k in range(L if B else 0):
                    p, c = _clt_source(k, L, d)
                    _product((q.data_ptr() + k * d, s.data_ptr() + k * d // 128 * t, L * d, t, B),
                             (wq + p * F * pitch + c, wsc + (p * pitch + c) // 128 * F, pitch, F, F), (L - k) * d,
                             dx.data_ptr() + k * F * dx.element_size(), _DT[g.dtype], L * F, None, dev, st)
            if w_dtypes:
                dWs = [torch.empty((l + 1, F, d), dtype=dt, device=dev) for l, dt in enumerate(w_dtypes)]
                for l, dW in enumerate(dWs):
                    _product((kept[0].data_ptr(), kept[1].data_ptr(), t, L * F, (l + 1) * F), (qt.data_ptr() + l * d * t, qs.data_ptr() + l * d, t, L * d, d), B,
                             dW.data_ptr(), _DT[dW.dtype], d, None, dev, st)
        return dx, dWs, db.view(L, d) if need_db else None
    q, s, qt, qs, db = ops8.pack8_raw(g.transpose(0, 1), _E4M3, need_dx or not w_dtypes, bool(w_dtypes), sums=need_db)
    if need_dx:
        dx = torch.empty((B, L * F), dtype=torch.float32, device=dev)
        for l in range(L - 1, -1, -1):                     # (the last layer reaches every column and writes; the others add)
            K = (l + 1) * F
            ops8.gemm8(ops8.Block8(q[l:l + 1], s[l:l + 1], B, d), ops8.Block8(ws[2 * l], ws[2 * l + 1], K, d), out=dx[:, :K].unsqueeze(0), accumulate=l != L - 1)
        dx = dx.view(B, L, F).to(g.dtype)
    if w_dtypes:
        x = ops8.Block8(kept[0], kept[1], L * F, B)
        dWs = [ops8.gemm8(x.first_rows((l + 1) * F), ops8.Block8(qt[l:l + 1], qs[l:l + 1], d, B), out_dtype=dt).view(l + 1, F, d) for l, dt in enumerate(w_dtypes)]
    return dx, dWs, db


@torch.library.custom_op("clt_hip::clt_decoder8", mutates_args=(), device_types=_DEV)
def _clt_decoder8_op(feat: Tensor, b: Optional[Tensor], Ws: List[Tensor], keep_x: bool, keep_w: bool) -> List[Tensor]:
    """-> [recons [B, L, d], the tensors kept for the backward pass]."""
    out, kept = _clt_forward(feat, b, Ws, keep_x, keep_w)
    return [out] + kept


@_clt_decoder8_op.register_fake
def _(feat, b, Ws, keep_x, keep_w):
    _clt_check(feat, b, Ws)
    B, L, F = feat.shape
    d = Ws[0].shape[2]
    return [feat.new_empty(B, L, d)] + [feat.new_empty(shape, dtype=torch.uint8) for shape in _clt_kept_shapes(B, L, F, d, keep_x, keep_w)]


@torch.library.custom_op("clt_hip::clt_decoder8_bwd", mutates_args=(), device_types=_DEV)
def _clt_decoder8_bwd(g: Tensor, kept: List[Tensor], F: int, has_x: bool, need_dx: bool, w_dtype: Optional[torch.dtype], need_db: bool) -> List[Tensor]:
    """-> [dfeat of g's type, db fp32 (empty where not asked for), dW_0, ..., dW_{L-1} (w_dtype None: none)]."""
    B, L, d = g.shape
    shapes = _clt_kept_shapes(B, L, F, d, has_x, need_dx)
    if [tuple(t.shape) for t in kept[:len(shapes)]] != shapes or any(t.dtype != torch.uint8 or not t.is_contiguous() or t.device != g.device for t in kept):
        raise ValueError("`kept` is not what clt_decoder8 kept for this gradient")
    if w_dtype is not None and not has_x:
        raise ValueError("the weights' gradient needs the features that clt_decoder8 keeps with keep_x")
    _check_type(w_dtype)
    dx, dWs, db = _clt_gradients(g, kept, F, has_x, need_dx, [w_dtype] * L if w_dtype is not None else [], need_db)
    return [g.new_empty(0) if t is None else t for t in (dx, db)] + (dWs or [])


@_clt_decoder8_bwd.register_fake
def _(g, kept, F, has_x, need_dx, w_dtype, need_db):
    B, L, d = g.shape
    f32 = torch.float32
    out = [g.new_empty((B, L, F)) if need_dx else g.new_empty(0), g.new_empty((L, d), dtype=f32) if need_db else g.new_empty(0)]
    return out + [g.new_empty((l + 1, F, d), dtype=w_dtype) for l in range(L if w_dtype is not None else 0)]


def _clt_setup(ctx, inputs, output):
    feat, b, Ws, ctx.keep_x, ctx.keep_w = inputs
    ctx.F, ctx.w_dtype, ctx.b = feat.shape[2], Ws[0].dtype, None if b is None else (b.dtype, b.shape)
    ctx.save_for_backward(*output[1:])


def _clt_backward(ctx, grads):
    need_x, need_b, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1], any(ctx.needs_input_grad[2])
    if (need_w and not ctx.keep_x) or (need_x and not ctx.keep_w):
        raise RuntimeError("clt_decoder8 was called without keeping what this gradient needs (keep_x for dW, keep_w for the features')")
    dx, db, *dWs = torch.ops.clt_hip.clt_decoder8_bwd(grads[0], list(ctx.saved_tensors), ctx.F, ctx.keep_x, need_x, ctx.w_dtype if need_w else None, need_b)
    # (a list argument's gradients are a list, of None where none is asked for)
    return dx if need_x else None, db.to(ctx.b[0]).reshape(ctx.b[1]) if need_b else None, list(dWs) if need_w else [None] * grads[0].shape[1], None, None


_clt_decoder8_op.register_autograd(_clt_backward, setup_context=_clt_setup)


class _CltDecoder8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feat, b, *Ws):
        need_w = any(ctx.needs_input_grad[2:])
        out, kept = _clt_forward(feat, b, Ws, need_w, ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        ctx.F, ctx.has_x, ctx.w_dtypes = feat.shape[2], need_w, [w.dtype for w in Ws]
        ctx.b = None if b is None else (b.dtype, b.shape)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        need = ctx.needs_input_grad
        dx, dWs, db = _clt_gradients(g, ctx.saved_tensors, ctx.F, ctx.has_x, need[0], ctx.w_dtypes if any(need[2:]) else [], need[1])
        dWs = [None] * len(ctx.w_dtypes) if dWs is None else [dW if n else None for dW, n in zip(dWs, need[2:])]
        return (dx, db.to(ctx.b[0]).reshape(ctx.b[1]) if need[1] else None, *dWs)


def clt_decoder8(feat: Tensor, b: Optional[Tensor], Ws: List[Tensor]) -> Tensor:
    """recons [B, L, d] from feat [B, L, F] and Ws[l] [l + 1, F, d], b [L, d] (`clt_hip::clt_decoder`'s arguments)."""
    if _dispatched(feat, b, *Ws):
        grad = torch.is_grad_enabled()
        return torch.ops.clt_hip.clt_decoder8(feat, b, list(Ws), grad and any(W.requires_grad for W in Ws), grad and feat.requires_grad)[0]
    if not torch.is_grad_enabled():
        return _clt_forward(feat, b, Ws, False, False)[0]
    return _CltDecoder8.apply(feat, b, *Ws)


#: names of the registered ops, for tests and introspection
REGISTERED8 = ("linear8", "linear8_bwd", "clt_decoder8", "clt_decoder8_bwd")
