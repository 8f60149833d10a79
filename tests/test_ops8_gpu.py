"""8-bit block-scaled operators (crosslayer_transcoder_amd/ops8.py, custom_ops8.py) against plain arithmetic in 64 bits.

Tolerances.  Packing is defined bit for bit: codes, scale bytes and restored values are compared for equality.  A product with
an fp32 result has exact products (bf16 holds 2^e x code) and K + 1 fp32 additions in some order, each off by at most one
unit of the last place (the matrix unit may truncate): |err| <= (K + 1) 2^-23 sum|a b| + 2^-23 |bias|.  With a 16-bit result
the unit keeps at least 13 bits below the largest product of a group of 16, so a group is off by less than 16 * 2^-13 of its
largest product, all groups by less than 2^-9 sum|a b|, and the result is rounded once (eps / 2)."""
import math

import pytest
import torch

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
gpu = pytest.mark.gpu


def up(n):
    return -(-n // 128) * 128


def held64(x, fmt="e4m3", tiles=False):
    """-> (values float64 [L, R, C], exponents int64 [L, C blocks, R]) from the definition, on the CPU."""
    x = x.detach().cpu().double()
    L, R, C = x.shape
    p = torch.zeros(L, up(R), up(C), dtype=torch.float64)
    p[:, :R, :C] = torch.where(torch.isfinite(x), x.abs(), torch.zeros((), dtype=torch.float64))
    top = p.view(L, up(R), up(C) // 128, 128).amax(3)
    if tiles:
        top = top.view(L, up(R) // 128, 128, -1).amax(2).repeat_interleave(128, 1)
    e = torch.full_like(top, -112.0)
    for k in range(-111, 122):                                   # the smallest exponent that reaches the maximum
        e = torch.where(top > LARGEST[fmt] * 2.0 ** (k - 1), torch.full_like(e, float(k)), e)
    e = e[:, :R]
    s = torch.exp2(e).repeat_interleave(128, 2)[:, :, :C]
    codes = (x / s).float().to(F8[fmt])                          # x 2^-e is exact in fp32 (or far below the smallest code)
    inf = torch.isinf(x)
    v = codes.double() * s
    v = torch.where(inf, torch.full_like(v, math.nan) if fmt == "e4m3" else x, v)
    return v, e.long().transpose(1, 2)


def same(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def rnd(*shape, seed=0, dtype=torch.float32, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:                                                   # magnitudes that differ from row to row and column to column
        x = x * torch.exp2(torch.randint(-12, 12, shape[:-1] + (1,), generator=g).float()) * torch.exp2(torch.randint(-3, 3, shape[-1:], generator=g).float())
    return x.to(dtype).cuda()


def check_block(q, x, fmt, tiles=False):
    from crosslayer_transcoder_amd import ops8
    v, e = held64(x, fmt, tiles)
    L, R, C = x.shape
    assert (q.batch, q.rows, q.cols, q.fmt) == (L, R, C, fmt)
    assert torch.equal(q.scale[:, :, :R].cpu().long() - 127, e)
    assert same(ops8.dequantize8(q), v)
    assert bool((q.data[:, :, C:] == 0).all())                   # the pad takes part in products


SHAPES = [(1, 1, 1), (1, 1, 127), (2, 16, 110), (1, 128, 128), (3, 129, 257), (1, 300, 1000), (2, 7, 2049), (1, 1000, 33), (12, 5, 768)]


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_packing_equals_the_definition(shape, dtype, fmt):
    from crosslayer_transcoder_amd import ops8
    x = rnd(*shape, seed=sum(shape), dtype=dtype)
    check_block(ops8.quantize8(x, fmt), x, fmt)
    check_block(ops8.quantize8_t(x, fmt), x.mT, fmt)
    q, qt = ops8.quantize8_both(x, fmt)
    check_block(q, x, fmt), check_block(qt, x.mT, fmt)
    w, wt = ops8.quantize8_tiles(x, fmt)
    check_block(w, x, fmt, tiles=True), check_block(wt, x.mT, fmt, tiles=True)
    assert same(ops8.dequantize8(w), ops8.dequantize8(wt).mT)
    for t in (torch.bfloat16, torch.float16):                    # restored values are rounded once
        assert same(ops8.dequantize8(q, t), held64(x, fmt)[0].float().to(t))


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_packing_at_the_borders(fmt):
    """Maxima at and next to largest * 2^e, zero blocks, subnormals, the largest floats, infinities and NaN."""
    from crosslayer_transcoder_amd import ops8
    x = torch.zeros(1, 24, 256)
    top = LARGEST[fmt]
    for r, m in enumerate([top, top * (1 + 2.0 ** -23), top * (1 - 2.0 ** -24), top * 2.0 ** -100, top * 2.0 ** -112, 2.0 ** -130, 2.0 ** -149, 3.0e38, 1.0, 0.0]):
        x[0, r, 3] = -m
        x[0, r, 4] = m / 3
        x[0, r, 200] = m
        x[0, r, 201] = m * 2.0 ** -9
    x[0, 10, 5], x[0, 10, 6], x[0, 10, 7] = math.inf, -math.inf, 2.5
    x[0, 11, 5], x[0, 11, 6] = math.nan, 0.1
    x[0, 12, :] = math.nan
    x[0, 13, :] = math.inf
    x[0, 14, :128] = torch.arange(128.0) / 16                    # ties of the rounding
    x[0, 15, :] = -0.0
    x = x.cuda()
    check_block(ops8.quantize8(x, fmt), x, fmt)
    check_block(ops8.quantize8_t(x, fmt), x.mT, fmt)
    w, wt = ops8.quantize8_tiles(x, fmt)
    check_block(w, x, fmt, tiles=True), check_block(wt, x.mT, fmt, tiles=True)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packing_of_views(dtype):
    """Token-major batches, slices that start anywhere, rows wider than the matrix, a transposed view, a broadcast row."""
    from crosslayer_transcoder_amd import ops8
    big = rnd(70, 3, 333, seed=5, dtype=dtype)
    for x in (big.transpose(0, 1), big[:, :, 1:300].transpose(0, 1), big[3:, 1:2, 7:].transpose(0, 1), big[:, :, :128].transpose(0, 1),
              big.permute(1, 2, 0), big[:1].expand(70, 3, 333).transpose(0, 1)):
        q, qt = ops8.quantize8_both(x)
        check_block(q, x, "e4m3"), check_block(qt, x.mT, "e4m3")
    check_block(ops8.quantize8(big[:, 1]), big[:, 1].unsqueeze(0), "e4m3")


@gpu
@pytest.mark.parametrize("shape", [(1, 1, 5), (2, 300, 130), (3, 128, 257), (1, 1000, 64)])
def test_column_sums(shape):
    """Sums of 128 rows in fp32, over the blocks in 64 bits: off by at most 128 additions' roundings and the last one."""
    from crosslayer_transcoder_amd import ops8
    x = rnd(*shape, seed=3)
    s = ops8.pack8_raw(x, 0, True, True, sums=True)[4].cpu().double()
    ref, mag = x.cpu().double().sum(1), x.cpu().double().abs().sum(1)
    assert bool(((s - ref).abs() <= 129 * 2.0 ** -24 * mag).all())


def values(q):
    from crosslayer_transcoder_amd import ops8
    return ops8.dequantize8(q).cpu().double()


def check_product(y, a, b, bias=None, base=None, whole=2.0 ** -20):
    """y [L, M, N] against the 64-bit product of the values held; whole: the tolerance of fp32 results' norm."""
    A, B = values(a), values(b)
    ref, mag = A @ B.mT, A.abs() @ B.abs().mT
    if bias is not None:
        ref, mag = ref + bias.cpu().double()[:, None], mag + bias.cpu().double().abs()[:, None]
    if base is not None:
        ref, mag = ref + base.cpu().double(), mag + base.cpu().double().abs()
    d = (y.cpu().double() - ref).abs()
    if y.dtype == torch.float32:
        bound = (a.cols + 2) * 2.0 ** -23 * mag
    else:
        fi = torch.finfo(y.dtype)
        bound = 2.0 ** -9 * mag + fi.eps / 2 * (ref.abs() + 2.0 ** -9 * mag) + fi.smallest_normal * fi.eps
    worst = float((d - bound).max())
    assert worst <= 0, worst
    # and as a whole: the alignment loss of normal data is about 2^-16, the rounding at most eps / 2 a value
    tol = whole if y.dtype == torch.float32 else torch.finfo(y.dtype).eps / 2 + 2.0 ** -12
    assert float(d.norm()) <= tol * float(ref.norm()) + 1e-30


PRODUCTS = [(1, 1, 1, 1), (1, 1, 110, 32), (2, 16, 110, 32), (1, 5, 768, 1000), (3, 33, 130, 257), (1, 128, 128, 128), (1, 200, 1000, 300),
            (2, 257, 513, 129), (1, 64, 4096, 96), (12, 3, 256, 64), (1, 300, 384, 512), (1, 100, 9000, 130), (2, 33, 20000, 15),
            (1, 130, 2048, 260), (1, 250, 2300, 77), (40, 100, 2500, 100)]


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", PRODUCTS)
def test_product(shape, out):
    from crosslayer_transcoder_amd import ops8
    L, M, K, N = shape
    a = ops8.quantize8(rnd(L, M, K, seed=1, spread=False))
    b = ops8.quantize8(rnd(L, N, K, seed=2, spread=False))
    bias = rnd(L, N, seed=3, spread=False)
    check_product(ops8.gemm8(a, b, out_dtype=out), a, b)
    check_product(ops8.gemm8(a, b, bias, out_dtype=out), a, b, bias)


#: enough 256 x 256 tiles to fill the chip: whole and partial ones, 1, 2, 3 and many blocks of k, odd rows of results
LARGE = [(1, 3000, 100, 2901), (12, 700, 256, 1100), (12, 701, 300, 1101), (3, 2048, 1024, 2048), (33, 300, 640, 515), (1, 128, 384, 40000),
         (1, 2100, 8192, 1801), (2, 1100, 12200, 1700), (1, 800, 24576, 1900), (2, 600, 20480, 1801),        # (these two: and K in slices)
         (1, 4100, 300, 4500), (3, 3000, 640, 2901),                # (and a rest of small tiles)
         (2, 2100, 300, 3501), (4, 1000, 640, 3900)]


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", LARGE)
def test_large_product(shape, out):
    from crosslayer_transcoder_amd import ops8
    L, M, K, N = shape
    a = ops8.quantize8(rnd(L, M, K, seed=1, spread=False), "e5m2" if K == 300 else "e4m3")
    b = ops8.quantize8(rnd(L, N, K, seed=2, spread=False), "e5m2" if K == 640 else "e4m3")
    bias = rnd(L, N, seed=3, spread=False)
    y = torch.full((M + 1, L, N), 7.0, dtype=out, device="cuda")
    ops8.gemm8(a, b, bias, out=y[:M].transpose(0, 1))
    check_product(y[:M].transpose(0, 1), a, b, bias)
    assert bool((y[M] == 7.0).all())
    if out == torch.float32:
        z = y[:M].transpose(0, 1).clone()
        ops8.gemm8(a, b, out=z, accumulate=True)
        check_product(z, a, b, base=y[:M].transpose(0, 1))


@gpu
def test_large_product_is_exact_on_integers_and_keeps_nan_in_its_row():
    from crosslayer_transcoder_amd import ops8
    g = torch.Generator().manual_seed(0)
    for (L, M, K, N) in [(1, 3000, 200, 3000), (5, 1000, 1000, 1500)]:
        a, b = torch.randint(-1, 2, (L, M, K), generator=g).float().cuda(), torch.randint(-1, 2, (L, N, K), generator=g).float().cuda()
        ref = a.cpu() @ b.cpu().mT
        f = torch.exp2(torch.randint(-20, 20, (L, M, 1), generator=g).float())                    # every row its own scale
        q, w = ops8.quantize8(a * f.cuda()), ops8.quantize8(b * 2.0 ** -30)
        assert same(ops8.gemm8(q, w), ref * f * 2.0 ** -30)
        assert same(ops8.gemm8(q, w, out_dtype=torch.bfloat16), (ref * f * 2.0 ** -30).bfloat16())
        a[0, 777, 5] = math.nan
        for out in (torch.float32, torch.bfloat16):
            bad = ops8.gemm8(ops8.quantize8(a), w, out_dtype=out).isnan()
            assert bool(bad[0, 777].all()) and int(bad.sum()) == N


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fa,fb", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
def test_product_of_the_wide_format(fa, fb, out):
    from crosslayer_transcoder_amd import ops8
    a, b = ops8.quantize8(rnd(2, 70, 300, seed=1, spread=False), fa), ops8.quantize8(rnd(2, 90, 300, seed=2, spread=False), fb)
    check_product(ops8.gemm8(a, b, out_dtype=out), a, b)


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_product_with_scales_far_apart(out):
    """Every row and block has its own scale: blocks differ by 2^24, rows by 2^24."""
    from crosslayer_transcoder_amd import ops8
    x, w = rnd(1, 50, 640, seed=1), rnd(1, 70, 640, seed=2)
    f = torch.exp2(torch.tensor([0.0, 12.0, -12.0, 3.0, -5.0])).repeat_interleave(128).cuda()
    a, b = ops8.quantize8(x * f), ops8.quantize8(w)
    A, B = values(a), values(b)
    ref, mag = A @ B.mT, A.abs() @ B.abs().mT
    d = (ops8.gemm8(a, b, out_dtype=out).cpu().double() - ref).abs()
    assert bool((d <= (642 * 2.0 ** -23 * mag if out == torch.float32 else 2.0 ** -9 * mag + 2.0 ** -8 * (ref.abs() + 2.0 ** -9 * mag))).all())


@gpu
def test_integers_multiply_exactly():
    """Small integers are held exactly and their sums stay below 2^11: every path gives the exact product, to the bit."""
    from crosslayer_transcoder_amd import ops8
    g = torch.Generator().manual_seed(0)
    for (L, M, K, N) in [(1, 1, 128, 64), (2, 130, 300, 270), (1, 300, 129, 515), (1, 17, 700, 33), (1, 600, 256, 600)]:
        a, b = torch.randint(-1, 2, (L, M, K), generator=g).float().cuda(), torch.randint(-1, 2, (L, N, K), generator=g).float().cuda()
        for fa in F8:
            q, w = ops8.quantize8(a, fa), ops8.quantize8(b)
            ref = a.cpu().double() @ b.cpu().double().mT
            assert same(ops8.gemm8(q, w), ref) and same(ops8.gemm8(q, w, out_dtype=torch.float16), ref)


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.float16])
def test_product_into_a_view_leaves_the_rest(out):
    """Token-major results [M, L, N] inside a wider buffer; what is not the result keeps its values."""
    from crosslayer_transcoder_amd import ops8
    for M, N, pad in ((37, 50, 3), (130, 256, 8), (300, 520, 0)):
        a, b = ops8.quantize8(rnd(3, M, 200, seed=1, spread=False)), ops8.quantize8(rnd(3, N, 200, seed=2, spread=False))
        buf = torch.full((M + 2, 3, N + pad + 1), 7.0, dtype=out, device="cuda")
        view = buf[1:M + 1, :, 1:N + 1].transpose(0, 1)
        ops8.gemm8(a, b, out=view)
        check_product(view, a, b)
        rest = buf.clone()
        rest[1:M + 1, :, 1:N + 1] = 7.0
        assert bool((rest == 7.0).all())


@gpu
def test_accumulate_and_empty_sizes():
    from crosslayer_transcoder_amd import ops8
    a, b = ops8.quantize8(rnd(2, 70, 300, seed=1, spread=False)), ops8.quantize8(rnd(2, 90, 300, seed=2, spread=False))
    base = rnd(2, 70, 90, seed=4, spread=False)
    out = base.clone()
    ops8.gemm8(a, b, out=out, accumulate=True)
    check_product(out, a, b, base=base)
    bias = rnd(2, 90, seed=6, spread=False)
    empty = ops8.quantize8(torch.zeros(2, 70, 0, device="cuda")), ops8.quantize8(torch.zeros(2, 90, 0, device="cuda"))
    assert same(ops8.gemm8(*empty, bias), bias[:, None].expand(2, 70, 90))             # no contraction: the bias alone
    assert bool((ops8.gemm8(*empty, out_dtype=torch.bfloat16) == 0).all())
    none = ops8.quantize8(torch.zeros(2, 0, 300, device="cuda"))
    assert ops8.gemm8(none, b).shape == (2, 0, 90) and ops8.gemm8(a, none).shape == (2, 70, 0)
    assert ops8.linear8(torch.zeros(0, 2, 300, device="cuda"), b).shape == (0, 2, 90)
    assert ops8.dequantize8(none).shape == (2, 0, 300)
    t = ops8.quantize8_t(torch.zeros(2, 0, 300, device="cuda"))
    assert (t.rows, t.cols) == (300, 0) and ops8.dequantize8(t).shape == (2, 300, 0)


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_nan_and_infinity_stay_in_their_rows(out):
    from crosslayer_transcoder_amd import ops8
    x = rnd(1, 40, 300, seed=1, spread=False)
    x[0, 3, 17], x[0, 20, 299] = math.nan, math.inf
    b = ops8.quantize8(rnd(1, 50, 300, seed=2, spread=False))
    for fmt in F8:
        y = ops8.gemm8(ops8.quantize8(x, fmt), b, out_dtype=out)
        bad = ~torch.isfinite(y[0]).all(1)
        assert bad.nonzero().flatten().tolist() == [3, 20]
        assert not torch.isfinite(y[0, 3]).any()


LINEAR = [(1, 1, 768, 512), (1, 1, 8192, 96), (2, 2, 110, 32), (16, 1, 768, 1000), (17, 3, 200, 130), (32, 2, 768, 256), (33, 1, 513, 300), (64, 1, 1024, 64), (65, 2, 256, 70),
          (300, 1, 256, 640), (4, 1, 40000, 70), (1, 2, 33000, 33)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", LINEAR)
def test_linear_with_kept_weights(shape, dtype):
    from crosslayer_transcoder_amd import ops8
    T, L, K, N = shape
    x = rnd(T, L, K, seed=1, dtype=dtype, spread=False)
    w, _ = ops8.quantize8_tiles(rnd(L, N, K, seed=2, spread=False))
    bias = rnd(L, N, seed=3, spread=False)
    q = ops8.quantize8(x.transpose(0, 1))
    for out in (None, torch.float32):
        y = ops8.linear8(x, w, bias, out_dtype=out)
        assert y.shape == (T, L, N) and y.dtype == (out or dtype)
        check_product(y.transpose(0, 1), q, w, bias)
    check_product(ops8.linear8(x, w).transpose(0, 1), q, w)
    if L == 1:
        assert same(ops8.linear8(x[:, 0], w, bias), ops8.linear8(x, w, bias)[:, 0])


@gpu
def test_linear_of_a_padded_batch_and_views():
    """Tokens cut out of a wider buffer at an odd offset; each token's result does not depend on its neighbours."""
    from crosslayer_transcoder_amd import ops8
    buf = rnd(40, 2, 333, seed=1, spread=False)
    w, _ = ops8.quantize8_tiles(rnd(2, 70, 301, seed=2, spread=False))
    x = buf[3:30, :, 5:306]
    y = ops8.linear8(x, w)
    assert same(y, ops8.linear8(x.contiguous(), w))
    check_product(y.transpose(0, 1), ops8.quantize8(x.transpose(0, 1)), w)
    one = torch.cat([ops8.linear8(x[t:t + 1], w) for t in range(x.shape[0])])
    assert float((one - y).abs().max()) <= 303 * 2.0 ** -22 * float((x.abs().amax() * 301 * 4))
    poisoned = x.clone()
    poisoned[5] = math.nan
    y2 = ops8.linear8(poisoned, w)
    keep = torch.arange(x.shape[0]) != 5
    assert same(y2[keep.cuda()], y[keep.cuda()]) and bool(y2[5].isnan().all())


def reference_training(x, W, b, dy, kn):
    """[y, dx, dW, db] in float64 from the values held, W [L, K, N] (kn) or [L, N, K]."""
    X, G = x.transpose(0, 1), dy.transpose(0, 1)
    w = held64(W, tiles=True)[0]
    w = w if kn else w.mT
    y = held64(X)[0] @ w + (b.cpu().double()[:, None] if b is not None else 0.0)
    xt, gt = held64(X.mT)[0], held64(G.mT)[0]
    dW = xt @ gt.mT
    return [y.transpose(0, 1), (held64(G)[0] @ w.mT).transpose(0, 1), dW if kn else dW.mT, dy.cpu().double().sum(0)]


def close(got, ref, tol):
    err = float((got.detach().cpu().double() - ref).norm())
    assert err <= tol * float(ref.norm()) + 1e-30, (err, float(ref.norm()))


TRAIN = [(1, 1, 1, 1), (16, 2, 110, 32), (130, 3, 257, 70), (64, 1, 768, 512), (5, 4, 40, 300), (300, 1, 128, 640)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", TRAIN)
def test_training_linear(shape, dtype):
    """Encoder and per-layer decoder, every gradient.  fp32: K (or T) roundings of 2^-23 at worst, of random sign; 16 bits: one
    rounding and the alignment loss."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    T, L, K, N = shape
    x = rnd(T, L, K, seed=1, dtype=dtype, spread=False).requires_grad_()
    b = rnd(L, N, seed=3, spread=False).requires_grad_()
    dy = rnd(T, L, N, seed=4, dtype=dtype, spread=False)
    W = (rnd(L, N, K, seed=2, spread=False) * 0.1).requires_grad_()
    for kn, f, Wp in ((False, lambda w: C.encoder8(x, w.permute(0, 2, 1), b), W),
                      (True, lambda w: C.plt_decoder8(x, w, b), W.detach().mT.contiguous().requires_grad_())):
        y = f(Wp)
        assert y.dtype == dtype
        dx, dW, db = torch.autograd.grad(y, (x, Wp, b), dy)
        assert dx.dtype == dtype and dW.dtype == torch.float32 and dW.shape == Wp.shape
        ref = reference_training(x, Wp, b, dy, kn)
        t = 2.0 ** -18 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 + 2.0 ** -12
        close(y, ref[0], t), close(dx, ref[1], t), close(dW, ref[2], 2.0 ** -18), close(db, ref[3], 2.0 ** -18)


@gpu
def test_gradients_equal_differences_where_nothing_is_rounded():
    """On integers the map is linear and every product exact: a gradient is the difference of two outputs, to the bit."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randint(-2, 3, s, generator=g).float().cuda()          # noqa: E731
    T, L, K, N = 9, 2, 130, 20
    x, W, b, dy = r(T, L, K), r(L, K, N), r(L, N), r(T, L, N)
    f = lambda x, W, b: float((C.plt_decoder8(x, W, b) * dy).double().sum())     # noqa: E731
    xg, Wg, bg = (t.clone().requires_grad_() for t in (x, W, b))
    (C.plt_decoder8(xg, Wg, bg) * dy).sum().backward()
    base = f(x, W, b)
    for t, grad, at in ((x, xg.grad, (3, 1, 129)), (x, xg.grad, (8, 0, 0)), (W, Wg.grad, (1, 128, 19)), (W, Wg.grad, (0, 5, 3)), (b, bg.grad, (1, 7))):
        old = float(t[at])
        t[at] = old + 1.0
        assert f(x, W, b) - base == float(grad[at])
        t[at] = old


@gpu
def test_only_what_is_needed_is_kept():
    """One byte an element of the input stays for the backward pass; without gradients nothing stays; W alone or x alone works."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, W, b = rnd(256, 2, 512, seed=1), rnd(2, 512, 128, seed=2), None
    out = torch.ops.clt_hip.linear8(x, W, b, True, True, False)
    assert out[1].numel() == x.numel() + x.numel() // 128
    for nx, nw in ((True, False), (False, True)):
        xi, Wi = x.clone().requires_grad_(nx), W.clone().requires_grad_(nw)
        C.plt_decoder8(xi, Wi, b).sum().backward()                                # (an expanded incoming gradient)
        assert (xi.grad is not None) == nx and (Wi.grad is not None) == nw
    with torch.no_grad():
        assert not C.plt_decoder8(x, W.requires_grad_(), b).requires_grad


@gpu
def test_empty_batch_gives_zero_gradients():
    from crosslayer_transcoder_amd import custom_ops8 as C
    x = torch.zeros(0, 2, 40, device="cuda", requires_grad=True)
    W, b = rnd(2, 40, 30).requires_grad_(), rnd(2, 30).requires_grad_()
    y = C.plt_decoder8(x, W, b)
    assert y.shape == (0, 2, 30)
    y.sum().backward()
    assert bool((W.grad == 0).all()) and bool((b.grad == 0).all()) and x.grad.shape == x.shape


@gpu
def test_opcheck():
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, b = rnd(9, 2, 40, seed=1, spread=False).requires_grad_(), rnd(2, 30, seed=2, spread=False).requires_grad_()
    W = rnd(2, 40, 30, seed=3, spread=False).requires_grad_()
    cases = {"linear8": (x, W, b, True, True, True)}
    kept = torch.ops.clt_hip.linear8(x.detach(), W.detach(), b.detach(), True, True, True)[1]
    cases["linear8_bwd"] = (rnd(9, 2, 30, seed=4, spread=False), kept, 40, True, True, True, torch.float32, True)
    Ws = [(rnd(l + 1, 40, 30, seed=5 + l, spread=False) * 0.2).requires_grad_() for l in range(2)]
    feat = torch.relu(x.detach()).requires_grad_()
    cases["clt_decoder8"] = (feat, b, Ws, True, True)
    kept = torch.ops.clt_hip.clt_decoder8(feat.detach(), b.detach(), [w.detach() for w in Ws], True, True)[1:]
    cases["clt_decoder8_bwd"] = (rnd(9, 2, 30, seed=4, spread=False), kept, 40, True, True, torch.float32, True)
    assert set(cases) == set(C.REGISTERED8)
    for name, args in cases.items():
        torch.library.opcheck(getattr(torch.ops.clt_hip, name).default, args)
    # sizes that are multiples of 128: the cross-layer decoder keeps its weights by source layer
    Ws = [(rnd(l + 1, 128, 128, seed=5 + l, spread=False) * 0.2).requires_grad_() for l in range(2)]
    feat = torch.relu(rnd(9, 2, 128, seed=1, spread=False)).requires_grad_()
    torch.library.opcheck(torch.ops.clt_hip.clt_decoder8.default, (feat, None, Ws, True, True))
    kept = torch.ops.clt_hip.clt_decoder8(feat.detach(), None, [w.detach() for w in Ws], True, True)[1:]
    torch.library.opcheck(torch.ops.clt_hip.clt_decoder8_bwd.default, (rnd(9, 2, 128, seed=4, spread=False), kept, 128, True, True, torch.float32, False))


@gpu
def test_captured_step_equals_eager_on_every_replay():
    """Forward and backward in one graph, replayed on changed inputs with eager work in between."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, W, b = rnd(70, 2, 130, seed=1).requires_grad_(), rnd(2, 130, 60, seed=2).requires_grad_(), rnd(2, 60, seed=3).requires_grad_()
    dy = rnd(70, 2, 60, seed=4)

    def step():
        y = C.plt_decoder8(x, W, b)
        return [y] + list(torch.autograd.grad(y, (x, W, b), dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(rnd(70, 2, 130, seed=10 + k)), dy.copy_(rnd(70, 2, 60, seed=20 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in out]
        assert all(torch.equal(u, v) for u, v in zip(got, step()))


@gpu
def test_two_streams_at_once():
    from crosslayer_transcoder_amd import ops8
    xs = [rnd(40 + 300 * i, 1, 700, seed=i, spread=False) for i in range(2)]
    ws = [ops8.quantize8_tiles(rnd(1, 500, 700, seed=5 + i, spread=False))[0] for i in range(2)]
    ref = [ops8.linear8(x, w) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                got[i].append(ops8.linear8(xs[i], ws[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref[i]) for i in range(2) for y in got[i])


@gpu
def test_captured_products_equal_eager_on_every_replay():
    """One graph with the few-token form and products whose K is cut (their workspaces share the graph's pool), replayed on changed inputs
    with eager calls of the same functions in between."""
    from crosslayer_transcoder_amd import ops8
    w, v = ops8.quantize8_weights(rnd(1, 70, 9000, seed=1, spread=False)), ops8.quantize8_weights(rnd(1, 1900, 20480, seed=2, spread=False))
    xs = [rnd(1, 9000, seed=10, spread=False), rnd(100, 9000, seed=11, spread=False), rnd(800, 20480, seed=12, dtype=torch.bfloat16, spread=False)]

    def calls():
        return [ops8.linear8(xs[0], w), ops8.linear8(xs[1], w), ops8.linear8(xs[2], v)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for k in range(4):
        for i, x in enumerate(xs):
            x.copy_(rnd(*x.shape, seed=20 + 3 * k + i, dtype=x.dtype, spread=False))
        expected = [y.clone() for y in calls()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected)), k


@gpu
def test_offsets_past_32_bits():
    """More than 2^31 elements in the input, the codes, the results and the weights: the last rows and columns."""
    from crosslayer_transcoder_amd import ops8
    R, C, last = 66000, 33000, 66000 // 128 * 128                                   # (last: first row of the last, partial block)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    q, t = ops8.quantize8_both(x)
    a, b = ops8.quantize8_both(x[last:])
    assert torch.equal(q.data[:, last:], a.data) and torch.equal(t.data[:, :, last:], b.data) and torch.equal(t.scale[:, -1], b.scale[:, -1])
    assert torch.equal(q.scale[:, :, last:R], a.scale[:, :, :R - last])
    assert same(ops8.dequantize8(q, torch.bfloat16)[:, last:], ops8.dequantize8(a, torch.bfloat16))
    del x, t, b
    m, n = q.first_columns(256), ops8.quantize8(rnd(1, C, 256, seed=1, spread=False))
    tail = ops8.Block8(n.data[:, C - 300:], n.scale[:, :, C - 300:], 300, 256)
    for dtype in (torch.bfloat16, torch.float32):
        y = ops8.gemm8(m, n, out_dtype=dtype)
        check_product(y[:, last:, C - 300:], a.first_columns(256), tail)
        del y
    del q, m
    K, N = 131072, 33000
    w = ops8.Block8(torch.randint(0, 100, (1, N, K), dtype=torch.uint8, device="cuda", generator=gen), torch.full((1, K // 128, N), 120, dtype=torch.uint8, device="cuda"), N, K)
    end = ops8.Block8(w.data[:, N - 64:], w.scale[:, :, N - 64:], 64, K)
    for T in (1, 40):
        v = rnd(T, K, seed=3, spread=False)
        # K additions one after another, each off by at most 2^-23 of the sum so far; sums of terms of random sign grow as sqrt(j / K) of
        # the last one, and errors of random sign add by squares: 2^-23 sqrt(sum_j j / K) = 2^-23 sqrt(K / 2) of the result's norm
        check_product(ops8.linear8(v, w)[None, :, N - 64:], ops8.quantize8(v), end, whole=2.0 ** -23 * math.sqrt(K / 2))


@gpu
def test_broadcast_inputs():
    """Tensors expanded over tokens or layers (strides of zero), as inputs and as gradients."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    from crosslayer_transcoder_amd import ops8
    x, W = rnd(1, 1, 300, seed=1, spread=False).expand(140, 2, 300), rnd(2, 300, 70, seed=2, spread=False)
    q, t = ops8.quantize8_both(x.transpose(0, 1))
    a, b = ops8.quantize8_both(x.transpose(0, 1).contiguous())
    assert torch.equal(q.data, a.data) and torch.equal(t.data, b.data) and torch.equal(t.scale, b.scale)
    w = ops8.quantize8_weights(W, transposed=True)
    assert same(ops8.linear8(x, w), ops8.linear8(x.contiguous(), w)) and same(ops8.linear8(x[:3], w), ops8.linear8(x[:3].contiguous(), w))
    leaves = [x.contiguous().requires_grad_(), W.clone().requires_grad_()]
    for dy in (torch.ones((), device="cuda").expand(140, 2, 70), rnd(1, 1, 70, seed=3, spread=False).expand(140, 2, 70), rnd(140, 1, 70, seed=4, spread=False).expand(140, 2, 70)):
        got = torch.autograd.grad(C.plt_decoder8(*leaves, None), leaves, dy)
        want = torch.autograd.grad(C.plt_decoder8(*leaves, None), leaves, dy.contiguous())
        assert all(torch.equal(u, v) for u, v in zip(got, want))


@gpu
def test_kept_bytes_that_do_not_fit_are_refused():
    x, W, dy = rnd(9, 2, 40, seed=1, spread=False), rnd(2, 40, 30, seed=2, spread=False), rnd(9, 2, 30, seed=3, spread=False)
    _, both = torch.ops.clt_hip.linear8(x, W, None, True, True, True)
    _, only_w = torch.ops.clt_hip.linear8(x, W, None, True, False, True)
    bwd = torch.ops.clt_hip.linear8_bwd
    assert torch.equal(bwd(dy, both, 40, True, True, True, None, False)[0], bwd(dy, only_w, 40, True, False, True, None, False)[0])
    for args in ((both[:-1], 40, True, True, True, None, False), (only_w, 40, True, True, True, None, False), (both.cpu(), 40, True, True, True, None, False),
                 (only_w, 40, True, False, True, torch.float32, False), (both.view(torch.int8), 40, True, True, True, None, False), (both, 400, True, True, True, None, False)):
        with pytest.raises((ValueError, RuntimeError)):
            bwd(dy, *args)


@gpu
@pytest.mark.parametrize("F,d", [(128, 128), (40, 30)])
def test_kept_tensors_that_do_not_fit_are_refused(F, d):
    feat, Ws, g = rnd(9, 2, F, seed=1, spread=False), [rnd(l + 1, F, d, seed=2 + l, spread=False) for l in range(2)], rnd(9, 2, d, seed=5, spread=False)
    kept = torch.ops.clt_hip.clt_decoder8(feat, None, Ws, True, True)[1:]
    only_w = torch.ops.clt_hip.clt_decoder8(feat, None, Ws, False, True)[1:]
    bwd = torch.ops.clt_hip.clt_decoder8_bwd
    assert torch.equal(bwd(g, kept, F, True, True, None, False)[0], bwd(g, only_w, F, False, True, None, False)[0])
    for args in ((kept, F + 128, True, True, None, False), (only_w, F, True, True, None, False), (kept[:2], F, True, True, None, False),
                 ([t.cpu() for t in kept], F, True, True, None, False), (only_w, F, False, True, torch.float32, False),
                 ([t.view(torch.int8) for t in kept], F, True, True, None, False)):
        with pytest.raises((ValueError, RuntimeError)):
            bwd(g, *args)


def reference_clt(feat, Ws, b, g):
    """[recons, dfeat, db, dW_l ...] of the cross-layer decoder in float64 from the values held."""
    B, L, F = feat.shape
    d = Ws[0].shape[2]
    flat = feat.detach().reshape(1, B, L * F)
    xt = held64(flat.mT)[0][0]                                                    # [L F, B]
    dfeat, recons, dWs = torch.zeros(B, L * F, dtype=torch.float64), [], []
    for l, W in enumerate(Ws):
        K = (l + 1) * F
        w = held64(W.detach().reshape(1, K, d), tiles=True)[0][0]
        recons.append(held64(flat[:, :, :K])[0][0] @ w + (b[l].detach().cpu().double() if b is not None else 0.0))
        dfeat[:, :K] += held64(g[:, l].unsqueeze(0))[0][0] @ w.mT
        dWs.append((xt[:K] @ held64(g[:, l].unsqueeze(0).mT)[0][0].mT).reshape(l + 1, F, d))
    return [torch.stack(recons, 1), dfeat.view(B, L, F), g.cpu().double().sum(0)] + dWs


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 3, 40, 30), (130, 2, 256, 70), (64, 4, 128, 110), (33, 1, 300, 64), (9, 1, 128, 128), (70, 3, 128, 128), (40, 4, 256, 384), (200, 5, 384, 128), (0, 3, 128, 128), (0, 2, 40, 30)])
def test_cross_layer_decoder(shape, dtype):
    """Dictionaries that are a multiple of 128 (one packing for all target layers) and not; outputs that are (the features' gradient is
    one product a source layer) and not (a sum of L products in fp32, rounded once); odd and even numbers of layers; no tokens."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    B, L, F, d = shape
    feat = torch.relu(rnd(B, L, F, seed=1, dtype=dtype, spread=False)).requires_grad_()
    Ws = [(rnd(l + 1, F, d, seed=2 + l, spread=False) * 0.1).requires_grad_() for l in range(L)]
    b, g = rnd(L, d, seed=9, spread=False).requires_grad_(), rnd(B, L, d, seed=10, dtype=dtype, spread=False)
    y = C.clt_decoder8(feat, b, Ws)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, [feat, b] + Ws, g)
    ref = reference_clt(feat, Ws, b, g)
    t = 2.0 ** -18 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 + 2.0 ** -12
    close(y, ref[0], t), close(grads[0], ref[1], t), close(grads[1], ref[2], 2.0 ** -18)
    for l in range(L):
        assert grads[2 + l].shape == Ws[l].shape
        close(grads[2 + l], ref[3 + l], 2.0 ** -18)
    z = torch.ops.clt_hip.clt_decoder8(feat, b, Ws, True, True)[0]
    assert torch.equal(y, z) and all(torch.equal(u, v) for u, v in zip(grads, torch.autograd.grad(z, [feat, b] + Ws, g)))


@gpu
@pytest.mark.parametrize("dec", ["clt", "plt"])
def test_modules_contract_in_8_bits(dec):
    """Encoder -> ReLU -> decoder as the modules run them under contractions8(): each stage against 64 bits on what it was given, the
    chain's gradients against the same formulas, a byte an element of every input kept, and the native forward untouched."""
    import crosslayer_transcoder_amd as cta
    from crosslayer_transcoder_amd.model import CrosslayerDecoder, CrossLayerTranscoder, Decoder, Encoder, ReLU
    L, d, F, B = 3, 96, 256, 64
    torch.manual_seed(1)
    m = CrossLayerTranscoder(ReLU(), Encoder(d, F, L), (CrosslayerDecoder if dec == "clt" else Decoder)(d, F, L)).cuda()
    x = rnd(B, L, d, seed=3, spread=False)
    native = m(x)[2].detach()
    with cta.contractions8():
        pre, feat, recons, _ = m(x)
    assert torch.equal(m(x)[2], native)
    g = rnd(B, L, d, seed=4, spread=False)
    feat.retain_grad(), pre.retain_grad()
    recons.backward(g)
    ref = reference_training(x, m.encoder.W.permute(0, 2, 1), m.encoder.b, pre.grad, False)
    close(pre.detach(), ref[0], 2.0 ** -18), close(m.encoder.W.grad.permute(0, 2, 1), ref[2], 2.0 ** -18), close(m.encoder.b.grad, ref[3], 2.0 ** -18)
    Ws = m.decoder.weights()
    if dec == "clt":
        ref = reference_clt(feat, Ws, m.decoder.b, g)
        grads = [m.decoder.b.grad] + [w.grad for w in Ws]
        close(recons.detach(), ref[0], 2.0 ** -18), close(feat.grad, ref[1], 2.0 ** -18)
        for got, want in zip(grads, ref[2:]):
            close(got, want, 2.0 ** -18)
    else:
        ref = reference_training(feat, m.decoder.W, m.decoder.b, g, True)
        for got, want in zip((recons.detach(), feat.grad, m.decoder.W.grad, m.decoder.b.grad), ref):
            close(got, want, 2.0 ** -18)
    assert same(pre.grad, torch.where(pre > 0, feat.grad, torch.zeros_like(feat.grad)))
    assert not torch.equal(recons, native)                                           # (the 8-bit path is what ran)


@gpu
@pytest.mark.parametrize("F,d", [(128, 128), (96, 64)])
def test_cross_layer_decoder_parts(F, d):
    """Each gradient alone equals the one computed with all of them; no gradient at all; a bias of another type."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    feat, b, g = torch.relu(rnd(20, 3, F, seed=1, spread=False)), rnd(3, d, seed=2, spread=False).half(), rnd(20, 3, d, seed=3, spread=False)
    Ws = [rnd(l + 1, F, d, seed=4 + l, spread=False) * 0.1 for l in range(3)]
    leaves = [feat, b] + Ws
    def grads(which):
        t = [u.detach().requires_grad_(i in which) for i, u in enumerate(leaves)]
        y = C.clt_decoder8(t[0], t[1], t[2:])
        return y, torch.autograd.grad(y, [t[i] for i in which], g) if which else ()
    y, full = grads(range(5))
    assert full[1].dtype == torch.float16
    for which in ([0], [1], [3], [0, 4], []):
        z, part = grads(which)
        assert torch.equal(y, z) and all(torch.equal(full[i], u) for i, u in zip(which, part))
    with torch.no_grad():
        assert torch.equal(C.clt_decoder8(*leaves[:2], leaves[2:]), y)
    c = torch.compile(lambda f, b, *w: C.clt_decoder8(f, b, list(w)), backend="aot_eager")(*(u.detach().requires_grad_() for u in leaves))
    assert torch.equal(c, y)


@gpu
def test_layers_with_packed_weights():
    """forward_layer(packed=pack8()): one token and a batch, every layer, encoder and both decoders."""
    from crosslayer_transcoder_amd import ops8
    from crosslayer_transcoder_amd.model import CrosslayerDecoder, Decoder, Encoder
    L, d, F = 3, 96, 200
    torch.manual_seed(2)
    enc, clt, plt = Encoder(d, F, L).cuda(), CrosslayerDecoder(d, F, L).cuda(), Decoder(d, F, L).cuda()
    for mod in (enc, clt, plt):
        torch.nn.init.normal_(mod.b)
    pe, pc, pp = enc.pack8(), clt.pack8(), plt.pack8()
    assert pe.nbytes() <= enc.W.numel() * 1.4                                       # (rows of 96 are held as 128)
    for shape in ((1, 1), (2, 3), (5, 40)):
        for l in range(L):
            x = rnd(*shape, d, seed=l, dtype=torch.bfloat16, spread=False)
            y = enc.forward_layer(x, l, packed=pe)
            assert y.shape == (*shape, F) and y.dtype == torch.bfloat16
            check_product(y.reshape(1, -1, F), ops8.quantize8(x.reshape(1, -1, d)), pe.of_batch(l), enc.b[l:l + 1])
            f = torch.relu(rnd(*shape, l + 1, F, seed=l, spread=False))
            z = clt.forward_layer(f, l, packed=pc)
            check_product(z.reshape(1, -1, d), ops8.quantize8(f.reshape(1, -1, (l + 1) * F)), pc[l], clt.b[l:l + 1])
            f = torch.relu(rnd(*shape, L, F, seed=l, spread=False))
            z = plt.forward_layer(f, l, packed=pp)
            check_product(z.reshape(1, -1, d), ops8.quantize8(f[:, :, l].reshape(1, -1, F)), pp.of_batch(l), plt.b[l:l + 1])


def test_results_that_share_elements_are_refused():
    from crosslayer_transcoder_amd.ops8 import _separate
    t = torch.empty(400)
    for good in (t[:24].view(2, 3, 4), t[:24].view(3, 2, 4).transpose(0, 1), t[:40].view(2, 4, 5)[:, :3, :4], t[:4].view(1, 1, 4), t[:6].view(6, 1, 1), t.as_strided((1, 1, 4), (0, 0, 1))):
        assert _separate(good), (good.shape, good.stride())
    for bad in (t[:4].view(1, 1, 4).expand(2, 1, 4), t[:12].view(1, 3, 4).expand(2, 3, 4), t.as_strided((2, 3, 4), (4, 4, 1)), t.as_strided((2, 3, 4), (12, 3, 1)),
                t.as_strided((1, 3, 4), (12, 4, 2)), t.as_strided((3, 2, 4), (4, 8, 1))):
        assert not _separate(bad), (bad.shape, bad.stride())


# ---- refusals (host checks: they run on the CPU) -----------------------------------------------------------------------------
def cpu_block(L, R, C, fmt="e4m3"):
    from crosslayer_transcoder_amd.ops8 import Block8
    return Block8(torch.zeros(L, R, up(C), dtype=torch.uint8), torch.zeros(L, up(C) // 128, up(R), dtype=torch.uint8), R, C, fmt)


def test_refusals_of_tensors():
    from crosslayer_transcoder_amd import ops8
    for f in (ops8.quantize8, ops8.quantize8_t, ops8.quantize8_both, ops8.quantize8_tiles):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops8.linear8(torch.zeros(4, 4), cpu_block(1, 3, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops8.gemm8(cpu_block(1, 3, 4), cpu_block(1, 3, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops8.dequantize8(cpu_block(1, 3, 4))
    with pytest.raises(TypeError):
        ops8.dequantize8(cpu_block(1, 3, 4), torch.float64)
    with pytest.raises(TypeError):
        ops8.dequantize8(torch.zeros(3, 4))


def test_refusals_of_block8():
    from crosslayer_transcoder_amd.ops8 import Block8
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8)                            # noqa: E731
    Block8(u(2, 5, 128), u(2, 1, 8), 5, 100)
    for args in ((u(2, 5, 128), u(2, 1, 4), 5, 100), (u(2, 5, 112), u(2, 1, 8), 5, 100), (u(2, 5, 128), u(2, 1, 8), 5, 129),
                 (u(2, 5, 128), u(1, 1, 8), 5, 100), (u(2, 4, 128), u(2, 1, 8), 5, 100), (u(5, 128), u(1, 8), 5, 100),
                 (u(2, 5, 128), u(2, 1, 5), 5, 100), (u(2, 5, 128), u(2, 1, 16)[:, :, 1:9], 5, 100),
                 (u(2, 128, 5).mT, u(2, 1, 8), 5, 100), (u(2, 5, 136)[:, :, :130], u(2, 1, 8), 5, 100), (u(2, 5, 256)[:, :, 1:129], u(2, 1, 8), 5, 100)):
        with pytest.raises(ValueError):
            Block8(*args)
    with pytest.raises(ValueError):
        Block8(u(2, 5, 128), u(2, 1, 8), 5, 100, "e3m4")
    with pytest.raises(TypeError):
        Block8(u(2, 5, 128).float(), u(2, 1, 8), 5, 100)
    q = Block8(u(2, 5, 384), u(2, 3, 128), 5, 300)
    assert q.first_rows(3).rows == 3 and q.first_columns(256).cols == 256 and q.of_batch(1).batch == 1
    assert q.columns(128, 128).cols == 128 and q.columns(256, 0).cols == 0 and q.columns(128, 172).cols == 172
    for bad in (lambda: q.first_rows(6), lambda: q.first_columns(200), lambda: q.first_columns(384), lambda: q.columns(64, 64), lambda: q.columns(128, 100),
                lambda: q.of_batch(2), lambda: q.of_batch(-1), lambda: q.columns(256, 128), lambda: q.columns(-128, 128), lambda: q.columns(128, -128)):
        with pytest.raises(ValueError):
            bad()


def test_refusals_of_the_library():
    """Arguments that the C entry points turn into errors before any launch."""
    from crosslayer_transcoder_amd._lib import lib
    p = 4096                                                                     # an aligned address nothing reads
    ok = dict(x=p, dt=0, rs=64, bs=0, b=1, r=4, c=64, f=0, t=0, q=p, s=p, qt=None, st=None, cs=None, ws=None, n=0)

    def pack(**k):
        a = {**ok, **k}
        return lib.clt_pack8(a["x"], a["dt"], a["rs"], a["bs"], a["b"], a["r"], a["c"], a["f"], a["t"], a["q"], a["s"], a["qt"], a["st"], a["cs"], a["ws"], a["n"], None)

    assert [pack(r=0), pack(c=-1), pack(b=0), pack(dt=3), pack(f=2), pack(s=None), pack(q=None, s=None), pack(x=None)] == [-1] * 8
    assert [pack(x=p + 2), pack(q=p + 8), pack(s=p + 1)] == [-4] * 3
    assert pack(cs=p, r=200) == -3 and pack(cs=p, r=200, ws=p, n=511) == -3

    def into(pitch=128, batch=0, qt=None, qt_pitch=0):
        return lib.clt_pack8_into(p, 0, 64, 0, 1, 4, 64, 0, 0, p, p, pitch, batch, 0, qt, qt, qt_pitch, 0, 0, None, None, 0, None)

    assert [into(pitch=64), into(qt=p), into(pitch=136), into(batch=8), into(qt=p, qt_pitch=132)] == [-1, -1, -4, -4, -4]

    def gemm(a=p, lda=128, ldas=128, b=p, ldb=128, ldbs=128, c=p, dt=0, ldc=64, M=4, N=4, K=100, batch=1, acc=0, fa=0, bias=None):
        return lib.clt_gemm8(a, p, fa, lda, ldas, 0, 0, b, p, 0, ldb, ldbs, 0, 0, c, dt, ldc, 0, bias, 0, M, N, K, batch, acc, None, 0, None)

    assert [gemm(M=0), gemm(N=0), gemm(K=-1), gemm(batch=0), gemm(dt=3), gemm(dt=1, acc=1), gemm(lda=112), gemm(ldbs=3), gemm(ldc=3), gemm(fa=2), gemm(c=None), gemm(a=None)] == [-1] * 12
    assert [gemm(a=p + 8), gemm(lda=136), gemm(c=p + 2), gemm(bias=p + 1), gemm(ldas=130)] == [-4] * 5
    assert gemm(K=5000, lda=5120, ldb=5120) == -3 and gemm(lda=1 << 24) == -6
    def fwd(x=p, dt=0, w=p, T=4, L=2, K=100, N=30, kx=1, kw=1, kept=p, ws=p, n=1 << 20):
        return lib.clt_linear8_forward(x, dt, 200, 100, w, 0, 100, 3000, 0, None, p, T, L, K, N, kx, kw, kept, ws, n, None)

    def bwd(dy=p, kept=p, T=4, N=30, dx=p, dw=p, db=p, ws=p, n=1 << 20):
        return lib.clt_linear8_backward(dy, 0, 60, 30, kept, 1, 0, T, 2, 100, N, dx, dw, 0, db, ws, n, None)

    assert [fwd(T=-1), fwd(L=0), fwd(K=0), fwd(N=0), fwd(x=p, w=None), fwd(dt=7, w=None)] == [-1] * 6
    assert [fwd(kept=None), fwd(kept=p + 8), fwd(ws=None), fwd(ws=p + 4), fwd(n=100)] == [-3] * 5
    assert fwd(T=0, kw=0) == 0                                                   # nothing to do
    assert [bwd(T=-1), bwd(N=0), bwd(dx=None, dw=None, db=None), bwd(dy=None)] == [-1] * 4
    assert [bwd(kept=None), bwd(ws=None), bwd(n=100)] == [-3] * 3
    assert lib.clt_linear8_kept_bytes(4, 2, 100, 30, 1, 1) == 2 * (100 * 128 + 128) * 2 and lib.clt_linear8_kept_bytes(4, 2, 100, 30, 0, 0) == 0
    assert lib.clt_unpack8(p, p, 0, 1, 4, 100, 112, 128, 0, 0, p, 0, None) == -1
    assert lib.clt_unpack8(p, p, 0, 1, 4, 100, 136, 128, 0, 0, p, 0, None) == -4


def test_refusals_of_the_training_ops():
    from crosslayer_transcoder_amd import custom_ops8 as C
    with pytest.raises(ValueError):
        C.plt_decoder8(torch.zeros(4, 2, 8), torch.zeros(2, 9, 3), None)
    with pytest.raises(ValueError):
        C.encoder8(torch.zeros(4, 2, 8), torch.zeros(3, 8, 3), None)
    with pytest.raises(ValueError):
        C.encoder8(torch.zeros(4, 8), torch.zeros(2, 8, 3), None)
    w = [torch.zeros(l + 1, 8, 3) for l in range(2)]
    for args in ((torch.zeros(4, 3, 8), None, w), (torch.zeros(4, 2, 9), None, w), (torch.zeros(4, 2, 8), torch.zeros(2, 4), w),
                 (torch.zeros(4, 2, 8), None, [w[0], w[1].double()]), (torch.zeros(4, 2, 8), None, w[::-1])):
        with pytest.raises(ValueError):
            C.clt_decoder8(*args)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        C.clt_decoder8(torch.zeros(4, 2, 8), None, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        C.plt_decoder8(torch.zeros(4, 2, 8), torch.zeros(2, 8, 3), None)


@gpu
def test_registered_op_equals_the_eager_function():
    """The dispatcher op (what torch.compile captures) and the eager autograd function give the same bits, forward and backward."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, W, b = (rnd(*s, seed=i, spread=False).requires_grad_() for i, s in enumerate(((40, 2, 130), (2, 130, 70), (2, 70))))
    dy = rnd(40, 2, 70, seed=9, spread=False)
    y = C.plt_decoder8(x, W, b)
    z = torch.ops.clt_hip.linear8(x, W, b, True, True, True)[0]
    assert torch.equal(y, z)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y, (x, W, b), dy), torch.autograd.grad(z, (x, W, b), dy)))
    c = torch.compile(lambda *t: C.plt_decoder8(*t), backend="aot_eager")(x, W, b)
    assert torch.equal(c, y)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(c, (x, W, b), dy), torch.autograd.grad(C.plt_decoder8(x, W, b), (x, W, b), dy)))
