"""8-bit block-scaled operators (include/clt_hip.h, "8-bit block-scaled matrices"): packing and restoring activations and
weights, products of packed matrices, and the linear map of a few or many tokens on kept packed weights.

A matrix [R, C] is held as 8-bit floats with one power-of-two scale for every row and block of 128 columns (`Block8`).
Tensors may be fp32, bf16 or fp16, of any size (zero rows included) and with any strides as long as the last dimension is
dense; everything runs on the tensors' device and on that device's current stream, allocates only through torch's caching
allocator and can be captured into a graph.  Nothing here is differentiable or seen by a tracer (make_fx, torch.jit.trace: refused):
custom_ops8.py is.  Non-HIP tensors raise: there is no fallback."""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch

from ._lib import CltError, lib

BLOCK = 128
FORMATS = {"e4m3": 0, "e5m2": 1}
#: tokens up to which linear8 streams the weights past all of them in one launch (clt_linear8_rows)
FEW_TOKENS = 32
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _up(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK * BLOCK


_tracing, _modes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack
_RECORDERS = (torch._C._TorchDispatchModeKey.PROXY, torch._C._TorchDispatchModeKey.FAKE, torch._C._TorchDispatchModeKey.FUNCTIONAL)


def _recorded():
    """Whether a tracer is taking down the calls around this one.  Inside the body of a registered op none is."""
    return _tracing() is not None or (_modes() > 0 and any(torch._C._get_dispatch_mode(k) is not None for k in _RECORDERS))


def _call(fn, *args):
    if _recorded():
        raise RuntimeError(f"{fn.__name__}: a tracer does not see launches on addresses; trace the functions of custom_ops8 or the modules' forward, "
                           "which are dispatcher ops")
    rc = fn(*args)
    if rc:
        raise CltError(fn.__name__, rc)


_HERE = contextlib.nullcontext()


def _on(device):
    """The tensors' device made current for a launch (a no-op when it is already)."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _fmt(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"8-bit format must be one of {sorted(FORMATS)}, got {fmt!r}")
    return FORMATS[fmt]


def _dense(x: torch.Tensor, dims=(2, 3)) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("crosslayer_transcoder_amd ops need CUDA (HIP) tensors; there is no CPU fallback")
    if x.dtype not in _DT:
        raise TypeError(f"expected float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() not in dims:
        raise ValueError(f"expected {' or '.join(map(str, dims))} dimensions, got shape {tuple(x.shape)}")
    return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


class Block8:
    """A batch of matrices [L, rows, cols] in 8 bits.  data: uint8 [L, rows, >= cols rounded up to 128], rows 16-byte aligned,
    codes of `fmt` ("e4m3" / "e5m2"), ZERO behind column `cols` up to the next multiple of 128; scale: uint8 [L, >= blocks of 128
    columns, >= rows], rows 4-byte aligned, byte e + 127 for the scale 2^e of a row's block.  The pack functions below make it; one may be
    built from kept tensors (a checkpoint of packed weights) as well, with e from -112 to 119 (e5m2: 112): there 2^e x code is exact in bf16,
    which products of fp32 or fp16 results and of few tokens rest on."""
    __slots__ = ("data", "scale", "rows", "cols", "fmt")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, rows: int, cols: int, fmt: str = "e4m3"):
        _fmt(fmt)
        if data.dtype is not torch.uint8 or scale.dtype is not torch.uint8:
            raise TypeError("codes and scale bytes are uint8 tensors")
        if data.device != scale.device:
            raise ValueError("codes and scale bytes are on different devices")
        shape, held = data.shape, scale.shape
        if len(shape) != 3 or len(held) != 3 or shape[0] != held[0]:
            raise ValueError("codes [L, rows, bytes] and scale bytes [L, blocks, rows] have three dimensions")
        wide = _up(cols)
        if rows < 0 or cols < 0 or shape[1] != rows or shape[2] < wide or held[1] < wide // BLOCK or held[2] < rows:
            raise ValueError(f"codes {tuple(shape)} / scale bytes {tuple(held)} do not hold a [{rows}, {cols}] matrix")
        (d0, d1, d2), (s0, s1, s2) = data.stride(), scale.stride()
        if data.numel() and (d2 != 1 or s2 != 1 or (d0 | d1 | data.data_ptr()) & 15 or (s0 | s1 | scale.data_ptr()) & 3):
            raise ValueError("packed rows are dense and start at multiples of 16 bytes (codes) and 4 bytes (scales)")
        self.data, self.scale, self.rows, self.cols, self.fmt = data, scale, rows, cols, fmt

    @classmethod
    def _made(cls, data, scale, rows, cols, fmt):
        """Of tensors that a pack function here made (the checks above are 2 us of a 10 us call)."""
        q = cls.__new__(cls)
        q.data, q.scale, q.rows, q.cols, q.fmt = data, scale, rows, cols, fmt
        return q

    @property
    def batch(self) -> int:
        return self.data.shape[0]

    @property
    def device(self):
        return self.data.device

    def first_rows(self, n: int) -> "Block8":
        """View of the first n rows."""
        if not 0 <= n <= self.rows:
            raise ValueError(f"{n} of {self.rows} rows")
        return Block8(self.data[:, :n], self.scale, n, self.cols, self.fmt)

    def first_columns(self, n: int) -> "Block8":
        """View of the first n columns, n a multiple of 128 (a block belongs to one contraction)."""
        return self.columns(0, n)

    def columns(self, start: int, n: int) -> "Block8":
        """View of n columns from `start`, a multiple of 128; n too unless they reach the last one."""
        if not 0 <= start <= start + n <= self.cols or start % BLOCK or (n % BLOCK and start + n != self.cols):
            raise ValueError(f"columns {start} .. {start + n} of {self.cols}: multiples of {BLOCK} are needed")
        return Block8(self.data[:, :, start:], self.scale[:, start // BLOCK:], self.rows, n, self.fmt)

    def of_batch(self, l: int) -> "Block8":
        """View of one matrix of the batch."""
        if not 0 <= l < self.batch:
            raise ValueError(f"matrix {l} of {self.batch}")
        return Block8(self.data[l:l + 1], self.scale[l:l + 1], self.rows, self.cols, self.fmt)

    def nbytes(self) -> int:
        return self.data.numel() + self.scale.numel()

    def __repr__(self):
        return f"Block8({self.fmt}, batch={self.batch}, rows={self.rows}, cols={self.cols})"


def _empty(x, rows, cols):
    """Unwritten codes and scale bytes of a [L, rows, cols] matrix (every byte of both is written by clt_pack8)."""
    L = x.shape[0]
    return (torch.empty((L, rows, _up(cols)), dtype=torch.uint8, device=x.device),
            torch.empty((L, _up(cols) // BLOCK, _up(rows)), dtype=torch.uint8, device=x.device))


def pack8_raw(x: torch.Tensor, fmt: int, along: bool, across: bool, tiles: bool = False, sums: bool = False):
    """clt_pack8 on x [L, R, C] -> (q, s, qt, st, column sums), None where not asked for."""
    L, R, C = x.shape
    q, s = _empty(x, R, C) if along else (None, None)
    qt, st = _empty(x, C, R) if across else (None, None)
    if L == 0 or R == 0 or C == 0:
        return q, s, qt, st, (torch.zeros((L, C), dtype=torch.float32, device=x.device) if sums else None)
    cs = ws = None
    nws = 0
    if sums:
        nws = lib.clt_pack8_sums_workspace_bytes(L, R, C)
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device)
        cs = torch.empty((L, C), dtype=torch.float32, device=x.device)
    with _on(x.device):
        _call(lib.clt_pack8, x.data_ptr(), _DT[x.dtype], x.stride(1), x.stride(0), L, R, C, fmt, int(tiles),
              q.data_ptr() if along else None, s.data_ptr() if along else None, qt.data_ptr() if across else None,
              st.data_ptr() if across else None, cs.data_ptr() if sums else None, ws.data_ptr() if sums else None, nws, _stream(x.device))
    return q, s, qt, st, cs


def _as3(x):
    x = _dense(x)
    return x.unsqueeze(0) if x.dim() == 2 else x


def quantize8(x: torch.Tensor, fmt: str = "e4m3") -> Block8:
    """x [R, C] or [L, R, C] held with blocks along its columns (the operand of a contraction over them)."""
    x = _as3(x)
    q, s, *_ = pack8_raw(x, _fmt(fmt), True, False)
    return Block8._made(q, s, x.shape[1], x.shape[2], fmt)


def quantize8_t(x: torch.Tensor, fmt: str = "e4m3") -> Block8:
    """x^T [C, R] held with blocks of 128 rows of x: the 8-bit checkpoint a contraction over the rows (a weight gradient) reads."""
    x = _as3(x)
    _, _, q, s, _ = pack8_raw(x, _fmt(fmt), False, True)
    return Block8._made(q, s, x.shape[2], x.shape[1], fmt)


def quantize8_both(x: torch.Tensor, fmt: str = "e4m3") -> Tuple[Block8, Block8]:
    """(quantize8(x), quantize8_t(x)) from one read of x."""
    x = _as3(x)
    q, s, qt, st, _ = pack8_raw(x, _fmt(fmt), True, True)
    return Block8._made(q, s, x.shape[1], x.shape[2], fmt), Block8._made(qt, st, x.shape[2], x.shape[1], fmt)


def quantize8_tiles(x: torch.Tensor, fmt: str = "e4m3") -> Tuple[Block8, Block8]:
    """A weight matrix and its transpose, one scale per 128 x 128 tile: both hold the same values."""
    x = _as3(x)
    q, s, qt, st, _ = pack8_raw(x, _fmt(fmt), True, True, tiles=True)
    return Block8._made(q, s, x.shape[1], x.shape[2], fmt), Block8._made(qt, st, x.shape[2], x.shape[1], fmt)


def quantize8_weights(x: torch.Tensor, transposed: bool = False, fmt: str = "e4m3") -> Block8:
    """One form of quantize8_tiles: a weight matrix [N, K] as linear8 and gemm8 contract it, or (transposed) a [K, N] one."""
    x = _as3(x)
    q, s, qt, st, _ = pack8_raw(x, _fmt(fmt), not transposed, transposed, tiles=True)
    return Block8._made(qt, st, x.shape[2], x.shape[1], fmt) if transposed else Block8._made(q, s, x.shape[1], x.shape[2], fmt)


def dequantize8(q: Block8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values held, [L, rows, cols], each rounded once to `dtype` (exact in fp32, and in bf16 for normal numbers)."""
    if dtype not in _DT:
        raise TypeError(f"expected float32, bfloat16 or float16, got {dtype}")
    _hip(q)
    out = torch.empty((q.batch, q.rows, q.cols), dtype=dtype, device=q.device)
    if out.numel():
        with _on(q.device):
            _call(lib.clt_unpack8, q.data.data_ptr(), q.scale.data_ptr(), FORMATS[q.fmt], q.batch, q.rows, q.cols, q.data.stride(1),
                  q.scale.stride(1), q.data.stride(0), q.scale.stride(0), out.data_ptr(), _DT[dtype], _stream(q.device))
    return out


def _hip(q):
    if not isinstance(q, Block8):
        raise TypeError("expected a Block8")
    if not q.data.is_cuda:
        raise RuntimeError("crosslayer_transcoder_amd ops need CUDA (HIP) tensors; there is no CPU fallback")


def _bias(bias, L, N, device):
    if bias is None:
        return None
    if bias.device != device or bias.numel() != L * N or (bias.dim() > 1 and tuple(bias.shape) != (L, N)):
        raise ValueError(f"bias must be [{L}, {N}] on the operands' device")
    if not bias.dtype.is_floating_point:
        raise TypeError(f"bias must be floating point, got {bias.dtype}")
    return bias if bias.dtype is torch.float32 and bias.is_contiguous() else bias.to(torch.float32).contiguous()


def _separate(out):
    """Whether the rows of out [L, M, N] are dense and no two of them share an element."""
    (L, M, N), (sb, sr, sc) = out.shape, out.stride()
    if (N > 1 and sc != 1) or (M > 1 and sr < N) or (L > 1 and sb < N):
        return False
    return L == 1 or M == 1 or sb >= (M - 1) * sr + N or sr >= (L - 1) * sb + N


def gemm8(a: Block8, b: Block8, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
          out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """out [L, M, N] (+)= a [L, M, K] @ b [L, N, K]^T + bias [L, N].  fp32 and fp16 results: exact products, fp32 sums, one rounding; bf16
    results: the 8-bit matrix instructions, at twice the rate.  These align the products of a group of 16 k to about 14 bits below the
    largest one: off by less than 2^-9 of the sum of |a b|, by about 1e-5 of the result's norm on normal data (rounding: 1.7e-3), more
    where large products cancel.  `out`: an [L, M, N] tensor or view with a dense last dimension to write into (its dtype counts), sharing
    nothing with the operands; accumulate: add to it (fp32 only).  The codes of a row of a or b take at most 8 MB."""
    _hip(a), _hip(b)
    L, M, N, K = a.batch, a.rows, b.rows, a.cols
    if b.batch != L or b.cols != K or b.device != a.device:
        raise ValueError(f"operands do not match: {a} and {b}")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the tensor to add to")
        if out_dtype not in _DT:
            raise TypeError(f"expected float32, bfloat16 or float16, got {out_dtype}")
        out = torch.empty((L, M, N), dtype=out_dtype, device=a.device)
    elif out.dtype not in _DT or (accumulate and out.dtype != torch.float32):
        raise TypeError(f"cannot {'add to' if accumulate else 'write'} {out.dtype}")
    elif tuple(out.shape) != (L, M, N) or out.device != a.device or (out.numel() and not _separate(out)):
        raise ValueError(f"out must be an [{L}, {M}, {N}] tensor of non-overlapping dense rows on the operands' device")
    bias = _bias(bias, L, N, a.device)
    if out.numel():
        nws = lib.clt_gemm8_workspace_bytes(M, N, K, L)
        ws = torch.empty(nws, dtype=torch.uint8, device=a.device) if nws else None
        with _on(a.device):
            _call(lib.clt_gemm8, a.data.data_ptr(), a.scale.data_ptr(), FORMATS[a.fmt], a.data.stride(1), a.scale.stride(1),
                  a.data.stride(0), a.scale.stride(0), b.data.data_ptr(), b.scale.data_ptr(), FORMATS[b.fmt], b.data.stride(1),
                  b.scale.stride(1), b.data.stride(0), b.scale.stride(0), out.data_ptr(), _DT[out.dtype], out.stride(1) if M > 1 else N,
                  out.stride(0), bias.data_ptr() if bias is not None else None, N, M, N, K, L, int(accumulate),
                  ws.data_ptr() if nws else None, nws, _stream(a.device))
    return out


def linear8(x: torch.Tensor, w: Block8, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y [T, L, N] = x [T, L, K] @ w^T + bias with kept packed weights w [L, N, K] (x [T, K] -> y [T, N] when L == 1): x is packed in
    e4m3 with blocks along K on the way.  out_dtype: x's by default.  Up to FEW_TOKENS the products are exact whatever the type, above
    that as gemm8's (K up to 8 M there): a token's bf16 results may differ between the two, mostly in the last place."""
    x = _dense(x)
    _hip(w)
    two = x.dim() == 2
    if two:
        x = x.unsqueeze(1)
    T, L, K = x.shape
    if L != w.batch or K != w.cols or x.device != w.device:
        raise ValueError(f"x {tuple(x.shape)} does not match {w}")
    dt = x.dtype if out_dtype is None else out_dtype
    if dt not in _DT:
        raise TypeError(f"expected float32, bfloat16 or float16, got {dt}")
    N = w.rows
    y = torch.empty((T, L, N), dtype=dt, device=x.device)
    if 0 < T <= FEW_TOKENS and K and N and L:
        bias = _bias(bias, L, N, x.device)
        nws = lib.clt_linear8_rows_workspace_bytes(T, L, N, K)
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws else None
        with _on(x.device):
            _call(lib.clt_linear8_rows, x.data_ptr(), _DT[x.dtype], x.stride(0), x.stride(1), w.data.data_ptr(), w.scale.data_ptr(),
                  FORMATS[w.fmt], w.data.stride(1), w.scale.stride(1), w.data.stride(0), w.scale.stride(0),
                  bias.data_ptr() if bias is not None else None, N, y.data_ptr(), _DT[dt], L * N, N, T, L, N, K,
                  ws.data_ptr() if nws else None, nws, _stream(x.device))
    elif T and K and N and L:                               # quantize8 and gemm8 on one buffer (a third of their host time)
        bias = _bias(bias, L, N, x.device)
        k, t = _up(K), _up(T)
        nws = lib.clt_gemm8_workspace_bytes(T, N, K, L)
        tmp = torch.empty(L * (T * k + k // BLOCK * t) + nws, dtype=torch.uint8, device=x.device)
        q = tmp.data_ptr()
        s = q + L * T * k
        with _on(x.device):
            st = _stream(x.device)
            _call(lib.clt_pack8, x.data_ptr(), _DT[x.dtype], x.stride(0), x.stride(1), L, T, K, 0, 0, q, s, None, None, None, None, 0, st)
            _call(lib.clt_gemm8, q, s, 0, k, t, T * k, k // BLOCK * t, w.data.data_ptr(), w.scale.data_ptr(), FORMATS[w.fmt], w.data.stride(1),
                  w.scale.stride(1), w.data.stride(0), w.scale.stride(0), y.data_ptr(), _DT[dt], L * N, N,
                  bias.data_ptr() if bias is not None else None, N, T, N, K, L, 0, s + L * (k // BLOCK) * t if nws else None, nws, st)
    else:
        gemm8(quantize8(x.transpose(0, 1)), w, bias, out=y.transpose(0, 1))
    return y.squeeze(1) if two else y
