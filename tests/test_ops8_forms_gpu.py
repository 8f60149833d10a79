"""8-bit block-scaled operators: every form that a product can take, and the calls next to the documented ones (the operators' own tests:
test_ops8_gpu.py).  Bounds are that file's; where every product and every partial sum is a whole number below 2^24, results are
compared to the bit."""
import math

import pytest
import torch

from tests.test_ops8_gpu import check_product, close, held64, reference_clt, reference_training, rnd, same, up, values

gpu = pytest.mark.gpu


def cancelling(L, R, K, seed):
    """Whole numbers of -1 .. 1 and, every 64 columns, two neighbours of 256: with weights_of below their products cancel, and a unit that
    aligns products to 14 bits below the largest of a few loses the small ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-1, 2, (L, R, K), generator=g).float()
    for k in range(0, K - 1, 64):
        x[:, :, k] = x[:, :, k + 1] = 256.0
    return x.cuda()


def weights_of(L, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-1, 2, (L, N, K), generator=g).float()
    for k in range(0, K - 1, 64):
        w[:, :, k], w[:, :, k + 1] = 256.0, -256.0
    return w.cuda()


#: small tiles, K in slices, large tiles, large tiles with a rest of small ones
CANCELLING = [(1, 200, 768, 300), (1, 100, 9000, 130), (1, 2048, 768, 8192), (1, 4100, 300, 4500), (1, 130, 128, 40000)]


@gpu
@pytest.mark.parametrize("shape", CANCELLING)
def test_fp16_and_fp32_results_keep_what_cancelling_products_leave(shape):
    """Sums below 2^11 are exact in fp16 and fp32; bf16 results stay within their documented bound."""
    from crosslayer_transcoder_amd import ops8
    L, M, K, N = shape
    a, b = cancelling(L, M, K, 1), weights_of(L, N, K, 2)
    ref = (a @ b.mT.contiguous()).cpu()                              # (exact: whole numbers, partial sums below 2^24)
    assert float(ref.abs().max()) <= 2048
    q, w = ops8.quantize8(a), ops8.quantize8(b)
    assert same(ops8.gemm8(q, w), ref) and same(ops8.gemm8(q, w, out_dtype=torch.float16), ref)
    assert same(ops8.linear8(a.transpose(0, 1).half(), w).transpose(0, 1), ref)
    y = ops8.gemm8(q, w, out_dtype=torch.bfloat16).cpu().float()
    assert bool(((y - ref).abs() <= 2.0 ** -9 * (a.abs() @ b.abs().mT.contiguous()).cpu() + 2.0 ** -8 * ref.abs()).all())


@gpu
def test_fp16_training_keeps_what_cancelling_products_leave():
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, w = cancelling(1, 300, 256, 1).transpose(0, 1).half(), weights_of(1, 384, 256, 2)
    y = C.encoder8(x, w.permute(0, 2, 1), None)
    assert same(y.transpose(0, 1), (x.transpose(0, 1).float() @ w.mT.contiguous()).cpu())
    # dx = g W^T: the gradient's neighbours of 256 meet +256 and -256 again
    g, W = cancelling(1, 300, 384, 3).transpose(0, 1).half(), weights_of(1, 256, 384, 4)             # W [L, K, N], blocks along N
    x = torch.zeros(300, 1, 256, dtype=torch.float16, device="cuda").requires_grad_()
    dx, = torch.autograd.grad(C.plt_decoder8(x, W, None), x, g)
    assert same(dx.transpose(0, 1), (g.transpose(0, 1).float() @ W.mT.contiguous()).cpu())


# ---- calls of the registered ops with tensors that do not fit: refused before any address is taken --------------------------------
def wrong_linear(t):
    """(x, W, b, kn) that do not belong together; t makes a tensor of a shape."""
    x = t(4, 2, 8)
    return [(x, t(1, 8, 3), None, True), (x, t(3, 8, 3), None, True), (x, t(2, 7, 3), None, True), (x, t(2, 3, 7), None, False), (x, t(2, 8, 3), None, False),
            (x, t(8, 3), None, True), (t(4, 8), t(2, 8, 3), None, True), (x, t(2, 8, 3), t(2, 4), True), (x, t(2, 8, 3), t(5), True), (x, t(2, 8, 3), t(3, 2), True)]


def wrong_clt(t):
    """(features, b, Ws): too many and too few matrices, one with more source layers, features or outputs than its place holds."""
    f = t(4, 2, 8)
    W = lambda *F: [t(l + 1, n, 3) for l, n in enumerate(F)]          # noqa: E731
    return [(f, None, W(8, 8, 8)), (f, None, W(8)), (f, None, []), (f, None, W(8, 9)), (f, None, W(9, 8)), (f, None, W(9, 9)), (f, None, [t(2, 8, 3), t(2, 8, 3)]),
            (f, None, [t(1, 8, 3), t(2, 8, 4)]), (f, None, [t(1, 8, 3), t(2, 24)]), (f, t(2, 4), W(8, 8)), (f, t(6), W(8, 8)), (t(4, 16), None, W(8, 8))]


@pytest.mark.parametrize("device", ["meta", "cpu", pytest.param("cuda", marks=gpu)])
def test_registered_ops_refuse_what_does_not_fit(device):
    """meta: what a tracer asks; cpu: the functions that the ops' bodies call; cuda: the ops themselves."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    t = lambda *s: torch.zeros(*s, device=device)                      # noqa: E731
    body = device == "cpu"
    for x, W, b, kn in wrong_linear(t):
        with pytest.raises(ValueError):
            C._forward(x, W, b, kn, True, True) if body else torch.ops.clt_hip.linear8(x, W, b, kn, True, True)
    for f, b, Ws in wrong_clt(t):
        with pytest.raises(ValueError):
            C._clt_forward(f, b, Ws, True, True) if body else torch.ops.clt_hip.clt_decoder8(f, b, Ws, True, True)
    if device != "cpu":                                               # what fits passes
        assert torch.ops.clt_hip.linear8(t(4, 2, 8), t(2, 8, 3), t(2, 3), True, True, True)[0].shape == (4, 2, 3)
        assert torch.ops.clt_hip.linear8(t(4, 2, 8), t(2, 3, 8), t(6), False, True, True)[0].shape == (4, 2, 3)
        assert torch.ops.clt_hip.clt_decoder8(t(4, 2, 8), t(2, 3), [t(1, 8, 3), t(2, 8, 3)], True, True)[0].shape == (4, 2, 3)


@gpu
def test_registered_ops_refuse_other_devices_and_types():
    t = lambda *s, **k: torch.zeros(*s, **{"device": "cuda", **k})     # noqa: E731
    ops = torch.ops.clt_hip
    for args in ((t(4, 2, 8), t(2, 8, 3, device="cpu"), None), (t(4, 2, 8), t(2, 8, 3), t(2, 3, device="cpu")), (t(4, 2, 8), t(2, 8, 3, dtype=torch.float64), None)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.linear8(*args, True, True, True)
    Ws = [t(1, 8, 3), t(2, 8, 3)]
    for args in ((t(4, 2, 8), None, [Ws[0], Ws[1].cpu()]), (t(4, 2, 8), t(2, 3, device="cpu"), Ws), (t(4, 2, 8), None, [Ws[0], Ws[1].half()])):
        with pytest.raises((ValueError, RuntimeError)):
            ops.clt_decoder8(*args, True, True)
    kept, kepts = ops.linear8(t(4, 2, 8), t(2, 8, 3), None, True, True, True)[1], ops.clt_decoder8(t(4, 2, 8), None, Ws, True, True)[1:]
    with pytest.raises(TypeError):
        ops.linear8_bwd(t(4, 2, 3), kept, 8, True, True, True, torch.float64, False)
    with pytest.raises(TypeError):
        ops.clt_decoder8_bwd(t(4, 2, 3), kepts, 8, True, True, torch.float64, False)


@gpu
@pytest.mark.parametrize("F,d", [(128, 128), (40, 30)])
def test_registered_cross_layer_decoder_with_some_gradients(F, d):
    """The op that torch.compile captures: each gradient alone (kept weights among them) equals the one of the eager function."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    leaves = [torch.relu(rnd(20, 2, F, seed=1, spread=False)), rnd(2, d, seed=2, spread=False)] + [rnd(l + 1, F, d, seed=3 + l, spread=False) * 0.1 for l in range(2)]
    g = rnd(20, 2, d, seed=9, spread=False)
    for which in ([0], [1], [2], [3], [0, 1], [0, 3], [2, 3], [0, 1, 2, 3]):
        got = []
        for f in (C.clt_decoder8, lambda feat, b, Ws: torch.ops.clt_hip.clt_decoder8(feat, b, Ws, any(i > 1 for i in which), 0 in which)[0]):
            t = [u.detach().clone().requires_grad_(i in which) for i, u in enumerate(leaves)]
            got.append(torch.autograd.grad(f(t[0], t[1], t[2:]), [t[i] for i in which], g))
        assert all(torch.equal(u, v) for u, v in zip(*got)), which
    c = torch.compile(lambda feat, b, *Ws: C.clt_decoder8(feat, b, list(Ws)), backend="aot_eager")
    feat = leaves[0].clone().requires_grad_()
    want = torch.autograd.grad(C.clt_decoder8(feat, leaves[1], leaves[2:]), feat, g)[0]
    assert torch.equal(torch.autograd.grad(c(feat, *leaves[1:]), feat, g)[0], want)


# ---- tracers and modes: the calls are dispatcher ops wherever something records them ---------------------------------------------
class Seen(torch.utils._python_dispatch.TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def tracing_cases(t):
    """name -> (function of the inputs, inputs, the op it has to show)."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    W, b, Ws = t(2, 130, 70), t(2, 70), [t(1, 130, 70), t(2, 130, 70)]
    enc = t(2, 70, 130).permute(0, 2, 1)
    return {"plt_decoder8": (lambda x: C.plt_decoder8(x, W, b), t(40, 2, 130), "clt_hip.linear8"),
            "encoder8": (lambda x: C.encoder8(x, enc, b), t(40, 2, 130), "clt_hip.linear8"),
            "clt_decoder8": (lambda x: C.clt_decoder8(x, b, Ws), t(40, 2, 130), "clt_hip.clt_decoder8")}


@pytest.mark.parametrize("name", ["plt_decoder8", "encoder8", "clt_decoder8"])
def test_traced_calls_are_dispatcher_ops(name):
    """With fake tensors, on the CPU: the graph holds the op, not the allocations around a launch."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x, op = tracing_cases(lambda *s: torch.zeros(*s))[name]
    with torch.no_grad():
        code = make_fx(f, tracing_mode="fake", _allow_non_fake_inputs=True)(x).code
    assert op in code, code


@gpu
@pytest.mark.parametrize("name", ["plt_decoder8", "encoder8", "clt_decoder8"])
def test_traced_calls_equal_eager_ones(name):
    """make_fx on real tensors, without and with gradients, and torch.jit.trace, run on other inputs; a dispatch mode sees the op."""
    from torch.fx.experimental.proxy_tensor import make_fx
    n = iter(range(100))
    f, x, op = tracing_cases(lambda *s: rnd(*s, seed=next(n), spread=False))[name]
    z = rnd(*x.shape, seed=50, spread=False)
    with torch.no_grad():
        want = f(z)
        for traced in (make_fx(f)(x), torch.jit.trace(f, (x,), check_trace=False)):
            assert torch.equal(traced(z), want)
    with Seen() as mode:
        assert torch.equal(f(z), want)
    assert any(op in s for s in mode.names), mode.names

    def both(x):
        y = f(x)
        return y.detach(), torch.autograd.grad(y.square().sum(), x)[0]

    x, z = x.requires_grad_(), z.requires_grad_()
    traced = make_fx(both)(x)
    assert op + "_bwd" in traced.code
    assert all(torch.equal(u, v) for u, v in zip(traced(z), both(z)))
    assert torch.equal(torch.jit.trace(f, (x,), check_trace=False)(z), f(z))


@gpu
def test_traced_model_equals_the_eager_one():
    import crosslayer_transcoder_amd as cta
    from torch.fx.experimental.proxy_tensor import make_fx
    from crosslayer_transcoder_amd.model import CrosslayerDecoder, CrossLayerTranscoder, Encoder, ReLU
    torch.manual_seed(0)
    m = CrossLayerTranscoder(ReLU(), Encoder(96, 256, 2), CrosslayerDecoder(96, 256, 2)).cuda()
    x, z = rnd(20, 2, 96, seed=1, spread=False), rnd(20, 2, 96, seed=2, spread=False)
    with cta.contractions8(), torch.no_grad():
        want = m(z)[2]
        assert torch.equal(make_fx(lambda x: m(x)[2])(x)(z), want)


@gpu
def test_functions_of_ops8_refuse_tracers():
    """They are no dispatcher ops: a trace would hold their allocations and nothing of what fills them."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from crosslayer_transcoder_amd import ops8
    from crosslayer_transcoder_amd.model import Encoder
    w = ops8.quantize8_weights(rnd(1, 70, 130, seed=1, spread=False))
    q = ops8.quantize8(rnd(1, 9, 130, seed=2, spread=False))
    enc = Encoder(130, 70, 1).cuda().requires_grad_(False)               # (torch.jit.trace takes no closed-over leaves)
    packed = enc.pack8()
    x = rnd(40, 130, seed=3, spread=False)
    calls = [lambda x: ops8.linear8(x, w), lambda x: ops8.linear8(x[:3], w), lambda x: ops8.quantize8(x).data, lambda x: ops8.quantize8_t(x).data,
             lambda x: ops8.quantize8_tiles(x)[0].data, lambda x: ops8.dequantize8(q) + x[0, 0], lambda x: ops8.gemm8(q, w) + x[0, 0],
             lambda x: enc.forward_layer(x, 0, packed=packed)]
    with torch.no_grad():
        for f in calls:
            want = f(x)
            for trace in (lambda: make_fx(f)(x), lambda: torch.jit.trace(f, (x,), check_trace=False)):
                with pytest.raises(RuntimeError, match="tracer"):
                    trace()
            with Seen():                                              # (a mode that only watches: nothing is recorded, nothing refused)
                assert torch.equal(f(x), want)
            assert torch.equal(torch.compile(f, backend="aot_eager")(x), want)


# ---- every form that the rules choose, asked of the rules themselves ------------------------------------------------------------------
DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FORMATS = [("e4m3", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")]


def gemm_plan(L, M, K, N, out):
    """-> (tiles of 256 x 256 that cover C, those the large form computes, slices of K)."""
    import ctypes
    from crosslayer_transcoder_amd._lib import lib
    plan = (ctypes.c_int64 * 3)()
    assert lib.clt_gemm8_plan(M, N, K, L, DT[out], N * L, plan) == 0
    return tuple(plan)


def rows_plan(T, L, K, N):
    """-> (blocks of k a slice, slices, row groups in hand, chunks of rows a block walks, blocks)."""
    import ctypes
    from crosslayer_transcoder_amd._lib import lib
    plan = (ctypes.c_int64 * 5)()
    assert lib.clt_linear8_rows_plan(T, L, N, K, plan) == 0
    return tuple(plan)


def check_large(y, a, b, bias=None, base=None, exact=None):
    """check_product's bounds with the 64-bit products on the GPU, a matrix at a time; fp16 results are exact up to the fp32 sums and one rounding."""
    from crosslayer_transcoder_amd import ops8
    fi = torch.finfo(y.dtype)
    exact = y.dtype != torch.bfloat16 if exact is None else exact
    for l in range(a.batch):
        A, B = ops8.dequantize8(a.of_batch(l))[0].double(), ops8.dequantize8(b.of_batch(l))[0].double().T.contiguous()
        ref, mag = A @ B, A.abs() @ B.abs()
        if bias is not None:
            ref, mag = ref + bias[l].double(), mag + bias[l].double().abs()
        if base is not None:
            ref, mag = ref + base[l].double(), mag + base[l].double().abs()
        d = (y[l].double() - ref).abs()
        lost = ((a.cols + 2) * 2.0 ** -23 if exact else 2.0 ** -9) * mag
        # one rounding of the sum as computed: half a step of its magnitude, of the smallest normal number's below that
        bound = lost if y.dtype == torch.float32 else lost + fi.eps / 2 * (ref.abs() + lost).clamp(min=fi.smallest_normal)
        assert float((d - bound).max()) <= 0, float((d - bound).max())
        # as a whole: fp32 sums of random sign stay below sqrt(K) 2^-23, aligned products below 2^-12, a rounding below half a step
        tol = math.sqrt(a.cols + 2) * 2.0 ** -23 if exact else 2.0 ** -12
        if y.dtype != torch.float32:
            tol += fi.eps / 2
        assert float(d.norm()) <= tol * float(ref.norm()) + 1e-30
        del A, B, ref, mag, d, bound


#: (L, M, K, N): whole and partial tiles; 1, 2 and 3 blocks of k, over which the staging of the next tiles runs ahead; many of them; slices;
#: a rest of small tiles
LARGE_FORMS = [(1, 4096, 128, 12288), (1, 4000, 100, 12201), (1, 4096, 256, 12288), (1, 4000, 300, 12201), (1, 4096, 4096, 12288), (1, 4000, 4100, 12201),
               (1, 800, 24576, 1900), (1, 4100, 4100, 4500)]


@gpu
@pytest.mark.parametrize("formats", FORMATS)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", LARGE_FORMS)
def test_large_form(shape, out, formats):
    """Three tiles and more a block of the large form, for every type of results and pair of formats, with a bias and added to."""
    from crosslayer_transcoder_amd import ops8
    L, M, K, N = shape
    tiles, large, slices = gemm_plan(L, M, K, N, out)
    if K == 24576:
        assert large == tiles and slices > 1
    elif (M, K) == (4100, 4100):
        assert 0 < large < tiles and slices == 1
    else:
        assert large == tiles >= 768 and slices == 1
    a = ops8.quantize8(rnd(L, M, K, seed=1, spread=False), formats[0])
    b = ops8.quantize8(rnd(L, N, K, seed=2, spread=False), formats[1])
    bias = rnd(L, N, seed=3, spread=False)
    y = ops8.gemm8(a, b, bias, out_dtype=out)
    check_large(y, a, b, bias)
    if out == torch.float32:
        z = y.clone()
        ops8.gemm8(a, b, out=z, accumulate=True)
        check_large(z, a, b, base=y)
    assert torch.equal(y, ops8.gemm8(a, b, bias, out_dtype=out))                 # (the order of the sums is fixed)


@gpu
@pytest.mark.parametrize("formats", FORMATS)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,sliced,many", [((3, 500, 300, 901), False, False), ((1, 100, 9000, 130), True, False), ((33, 300, 640, 515), False, True)])
def test_small_form(shape, sliced, many, out, formats):
    """Up to 256 tiles (one a CU), K in slices, more than 256 (two a CU)."""
    from crosslayer_transcoder_amd import ops8
    L, M, K, N = shape
    tiles, large, slices = gemm_plan(L, M, K, N, out)
    assert large == 0 and (slices > 1) == sliced and (-(-M // 128) * -(-N // 128) * L * slices > 256) == many, (tiles, large, slices)
    a, b = ops8.quantize8(rnd(L, M, K, seed=1, spread=False), formats[0]), ops8.quantize8(rnd(L, N, K, seed=2, spread=False), formats[1])
    bias = rnd(L, N, seed=3, spread=False)
    check_large(ops8.gemm8(a, b, bias, out_dtype=out), a, b, bias)


@gpu
def test_weight_gradient_of_a_short_batch():
    """Up to 128 tokens: one block of k, enough tiles for the large form."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    from crosslayer_transcoder_amd import ops8
    T, K, N = 70, 4096, 8192
    assert gemm_plan(1, K, T, N, torch.float32) == (512, 512, 1)
    x, W, dy = rnd(T, 1, K, seed=1, spread=False), (rnd(1, K, N, seed=2, spread=False) * 0.01).requires_grad_(), rnd(T, 1, N, seed=3, spread=False)
    dW, = torch.autograd.grad(C.plt_decoder8(x, W, None), W, dy)
    check_large(dW, ops8.quantize8_t(x.transpose(0, 1)), ops8.quantize8_t(dy.transpose(0, 1)))


#: (T, L, K, N) -> what the rule has to choose for them (blocks of k a slice >=, slices > 1, groups in hand, chunks > 1)
ROWS_FORMS = [((20, 12, 130, 32001), (1, False, 1, True)),       # 17 .. 32 tokens: blocks that walk several chunks of rows, the last one ragged
              ((32, 3, 130, 66001), (1, False, 1, True)),
              ((3, 12, 130, 50001), (1, False, 2, True)),        # up to 16 tokens: two row groups, several chunks
              ((9, 5, 1200, 130000), (10, False, 2, True)),      # the same with long rows
              ((32, 1, 9000, 200), (5, True, 1, False)),         # slices of 32 tokens
              ((17, 2, 20000, 33), (6, True, 1, False)),
              ((24, 12, 1300, 12345), (11, False, 1, True)),     # long slices of 17 .. 32 tokens: the loop in steps, one block a CU
              ((17, 12, 1500, 20001), (12, False, 1, True)),
              ((32, 4, 2000, 20000), (8, True, 1, True)),        # slices and chunks
              ((1, 4, 70000, 1000), (60, True, 1, False)),
              ((16, 1, 768, 1000), (6, False, 1, False))]


@gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("shape,form", ROWS_FORMS)
def test_few_token_forms(shape, form, fmt):
    from crosslayer_transcoder_amd import ops8
    T, L, K, N = shape
    slice_kb, slices, g, chunks, _ = rows_plan(T, L, K, N)
    assert slice_kb >= form[0] and (slices > 1, g, chunks > 1) == form[1:], (slice_kb, slices, g, chunks)
    x, bias = rnd(T, L, K, seed=1, spread=False), rnd(L, N, seed=3, spread=False)
    w = ops8.quantize8(rnd(L, N, K, seed=2, spread=False), fmt)
    y = ops8.linear8(x, w, bias)
    check_large(y.transpose(0, 1), ops8.quantize8(x.transpose(0, 1)), w, bias)
    z = ops8.linear8(x.half(), w, bias)
    check_large(z.transpose(0, 1), ops8.quantize8(x.half().transpose(0, 1)), w, bias)
    z = ops8.linear8(x.bfloat16(), w)
    check_large(z.transpose(0, 1), ops8.quantize8(x.bfloat16().transpose(0, 1)), w, exact=True)
    assert torch.equal(y, ops8.linear8(x, w, bias))


@gpu
@pytest.mark.parametrize("K,slices", [(301, False), (9000, True)])
def test_a_token_does_not_depend_on_its_batch(K, slices):
    """Each of 27 tokens by itself, against 64 bits (test_ops8_gpu.py compares only within a few percent); to the bit where neither call cuts K:
    the same products in the same order."""
    from crosslayer_transcoder_amd import ops8
    x, w = rnd(27, 2, K, seed=1, spread=False), ops8.quantize8_weights(rnd(2, 70, K, seed=2, spread=False))
    assert (rows_plan(27, 2, K, 70)[1] > 1) == slices and (rows_plan(1, 2, K, 70)[1] > 1) == slices
    y, one = ops8.linear8(x, w), torch.cat([ops8.linear8(x[t:t + 1], w) for t in range(27)])
    check_large(one.transpose(0, 1), ops8.quantize8(x.transpose(0, 1)), w)
    assert slices or torch.equal(one, y)


def test_plans_are_refused_for_no_sizes():
    import ctypes
    from crosslayer_transcoder_amd._lib import lib
    p = (ctypes.c_int64 * 5)()
    assert [lib.clt_gemm8_plan(0, 1, 1, 1, 0, 1, p), lib.clt_gemm8_plan(1, 2, 1, 1, 0, 1, p), lib.clt_gemm8_plan(1, 1, 1, 1, 3, 1, p), lib.clt_gemm8_plan(1, 1, 1, 1, 0, 1, None)] == [-1] * 4
    assert [lib.clt_linear8_rows_plan(0, 1, 1, 1, p), lib.clt_linear8_rows_plan(33, 1, 1, 1, p), lib.clt_linear8_rows_plan(1, 1, 1, 1, None)] == [-1] * 3
    # results whose rows lie more than 2^21 elements apart: small tiles
    assert lib.clt_gemm8_plan(4096, 12288, 4096, 1, 0, 12288, p) == 0 and p[1] == 768
    assert lib.clt_gemm8_plan(4096, 12288, 4096, 1, 0, 1 << 22, p) == 0 and p[1] == 0


# ---- the ends of the scales' range -----------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("shape", [(40, 300, 70), (1, 300, 70), (100, 9000, 130), (4096, 200, 8192)])
def test_smallest_codes_take_part_in_products(shape):
    """e5m2 at the smallest exponent: codes of 1 to 3 times 2^-16 times 2^-112, subnormal numbers in bf16 and fp32, against weights of 2^110: whole
    multiples of 2^-18, exact for every type of results."""
    from crosslayer_transcoder_amd import ops8
    M, K, N = shape
    g = torch.Generator().manual_seed(0)
    few = torch.rand(K, generator=g) < 300 / K                                   # (sums stay below 2^8 in bf16, 2^11 in fp16)
    i = torch.randint(-1, 2, (M, K), generator=g).float() * few
    i[:, ::7] *= 3
    w = torch.randint(-1, 2, (N, K), generator=g).float() * (torch.rand(K, generator=g) < 0.3)
    a, b = ops8.quantize8((i.double() * 2.0 ** -128).float().cuda(), "e5m2"), ops8.quantize8((w * 2.0 ** 110).cuda(), "e5m2")
    assert bool((a.scale == 15).all()) and same(ops8.dequantize8(a)[0], i.double() * 2.0 ** -128)
    ref = i.cuda() @ w.cuda().T.contiguous()                                     # (whole numbers)
    assert float(ref.abs().max()) <= 256
    for out in (torch.float32, torch.bfloat16, torch.float16):
        assert same(ops8.gemm8(a, b, out_dtype=out)[0], ref.cpu().double() * 2.0 ** -18), out
    x = (w[:M] if M <= N else w[:1].expand(M, K)) * 2.0 ** 110                   # the other way round: kept weights that are tiny
    want = x.cuda().div(2.0 ** 110) @ i.cuda().T.contiguous()
    assert same(ops8.linear8(x.cuda(), a), want.cpu().double() * 2.0 ** -18)


@gpu
def test_largest_numbers():
    """Up to the last magnitude that rounds down, values are finite and products exact; above it they are held as 2^128 and restored as infinities."""
    from crosslayer_transcoder_amd import ops8
    for fmt, below, held in (("e4m3", 1.9375 - 2.0 ** -23, 1.875), ("e5m2", 1.875 - 2.0 ** -23, 1.75)):
        x = torch.zeros(40, 128)
        x[:, 5], x[1, 5] = below * 2.0 ** 127, -below * 2.0 ** 127
        q = ops8.quantize8(x.cuda(), fmt)
        assert float(ops8.dequantize8(q)[0, 0, 5]) == held * 2.0 ** 127
        w = ops8.quantize8(torch.full((40, 128), 2.0 ** -120).cuda())
        for out in (torch.float32, torch.bfloat16, torch.float16):
            y = ops8.gemm8(q, w, out_dtype=out)[0]
            assert bool((y[0] == held * 128).all()) and bool((y[1] == -held * 128).all()), (fmt, out)
    x[0, 5] = torch.finfo(torch.float32).max
    for fmt in ("e4m3", "e5m2"):
        assert float(ops8.dequantize8(ops8.quantize8(x.cuda(), fmt))[0, 0, 5]) == math.inf


def test_refusals_of_the_few_token_call():
    from crosslayer_transcoder_amd._lib import lib
    p = 4096                                                                     # an aligned address nothing reads

    def rows(x=p, dt=0, w=p, ws=p, ldw=128, ldws=128, y=p, T=4, L=1, N=40, K=100, bias=None, buf=None, n=0):
        return lib.clt_linear8_rows(x, dt, 100, 0, w, ws, 0, ldw, ldws, 0, 0, bias, 0, y, 0, N, 0, T, L, N, K, buf, n, None)

    assert [rows(T=0), rows(L=0), rows(N=0), rows(K=0), rows(dt=3), rows(x=None), rows(w=None), rows(ws=None), rows(y=None), rows(ldw=112), rows(ldws=39)] == [-1] * 11
    assert [rows(x=p + 2), rows(w=p + 8), rows(ldw=136), rows(y=p + 1), rows(bias=p + 2)] == [-4] * 5
    assert rows(T=33) == -6                                                      # an error like any other, not a code of its own
    assert rows(K=40000, ldw=40064, N=40) == -3 and rows(K=40000, ldw=40064, N=40, buf=p, n=16) == -3


# ---- the operators together, as a program uses them ---------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_serving_chain_on_packed_weights(tokens):
    """Encoder layer by layer -> every sparsifier -> both decoders on kept weights, each stage on what the one before it gave (fp32, which the
    sparsifiers take)."""
    from crosslayer_transcoder_amd import ops8
    from crosslayer_transcoder_amd.model import BatchTopK, CrosslayerDecoder, Decoder, Encoder, PerLayerBatchTopK, PerLayerTopK, ReLU
    L, d, F = 3, 96, 256
    torch.manual_seed(3)
    enc, clt, plt = Encoder(d, F, L).cuda(), CrosslayerDecoder(d, F, L).cuda(), Decoder(d, F, L).cuda()
    pe, pc, pp = enc.pack8(), clt.pack8(), plt.pack8()
    x = rnd(1, tokens, L, d, seed=4, spread=False)
    for sparsifier in (ReLU(), PerLayerTopK(k=8), BatchTopK(k=8, e=0.1), PerLayerBatchTopK(k=8, e=0.1, n_layers=L)):
        feats = []
        for l in range(L):
            pre = enc.forward_layer(x[:, :, l], l, packed=pe)
            feats.append(sparsifier.cuda()(pre, l))
            assert feats[-1].shape == (1, tokens, F) and feats[-1].dtype == torch.float32
            stack = torch.stack(feats, 2)
            y = clt.forward_layer(stack, l, packed=pc)
            check_large(y, ops8.quantize8(stack.reshape(1, tokens, -1)), pc[l], clt.b[l:l + 1])
        y = plt.forward_layer(stack, 1, packed=pp)
        check_large(y, ops8.quantize8(stack[:, :, 1]), pp.of_batch(1), plt.b[1:2])


@gpu
@pytest.mark.parametrize("F,d", [(256, 128), (200, 96)])
def test_captured_cross_layer_step_equals_eager_on_every_replay(F, d):
    from crosslayer_transcoder_amd import custom_ops8 as C
    L, B = 3, 140
    feat, b, g = torch.relu(rnd(B, L, F, seed=1)).requires_grad_(), rnd(L, d, seed=2).requires_grad_(), rnd(B, L, d, seed=3)
    Ws = [rnd(l + 1, F, d, seed=4 + l, spread=False).requires_grad_() for l in range(L)]

    def step():
        y = C.clt_decoder8(feat, b, Ws)
        return [y] + list(torch.autograd.grad(y, [feat, b] + Ws, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            feat.copy_(torch.relu(rnd(B, L, F, seed=10 + k))), g.copy_(rnd(B, L, d, seed=20 + k)), Ws[1].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in out]
        assert all(torch.equal(u, v) for u, v in zip(got, step())), k


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_of_16_bits(dtype):
    """Weights and biases in 16 bits: gradients in their types, each rounded once (bf16 ones from aligned products)."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    T, L, K, N = 150, 2, 256, 128
    x, dy = rnd(T, L, K, seed=1, spread=False).requires_grad_(), rnd(T, L, N, seed=2, spread=False)
    W, b = rnd(L, K, N, seed=3, dtype=dtype, spread=False).requires_grad_(), rnd(L, N, seed=4, dtype=dtype, spread=False).requires_grad_()
    y = C.plt_decoder8(x, W, b)
    dx, dW, db = torch.autograd.grad(y, (x, W, b), dy)
    assert (y.dtype, dx.dtype, dW.dtype, db.dtype) == (torch.float32, torch.float32, dtype, dtype)
    ref, t = reference_training(x, W, b, dy, True), torch.finfo(dtype).eps / 2 + 2.0 ** -12
    close(y.detach(), ref[0], 2.0 ** -18), close(dx, ref[1], 2.0 ** -18), close(dW, ref[2], t), close(db, ref[3], t)
    feat, Ws = torch.relu(x.detach()).requires_grad_(), [rnd(l + 1, K, N, seed=5 + l, dtype=dtype, spread=False).requires_grad_() for l in range(L)]
    y = C.clt_decoder8(feat, b, Ws)
    grads, ref = torch.autograd.grad(y, [feat, b] + Ws, dy), reference_clt(feat, Ws, b, dy)
    close(grads[0], ref[1], 2.0 ** -18), close(grads[1], ref[2], t)
    for dW, want in zip(grads[2:], ref[3:]):
        assert dW.dtype == dtype
        close(dW, want, t)


@gpu
@pytest.mark.parametrize("F,d", [(256, 128), (200, 96)])
def test_cross_layer_decoder_of_views(F, d):
    """Weights cut out of wider buffers, transposed ones, features and gradients with other strides: the bits of dense tensors."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    L, B = 3, 40
    feat, g = torch.relu(rnd(L, B, F + 5, seed=1, spread=False)), rnd(B, d, L, seed=2, spread=False)
    wide = [rnd(l + 2, F + 3, d + 7, seed=4 + l, spread=False) for l in range(L)]
    views = [wide[0][1:, 2:F + 2, 3:d + 3], wide[1][:2, :F, :d], rnd(3, d, F, seed=9, spread=False).mT]
    f, h = feat[:, :, 1:F + 1].transpose(0, 1), g.transpose(1, 2)
    got = []
    for dense in (False, True):
        t = [(u.contiguous() if dense else u).detach().requires_grad_() for u in (f, *views)]
        y = C.clt_decoder8(t[0], None, t[1:])
        got.append([y] + list(torch.autograd.grad(y, t, h.contiguous() if dense else h)))
    assert all(torch.equal(u, v) for u, v in zip(*got))


@gpu
def test_the_same_tensor_twice_and_a_stream_of_its_own():
    """One leaf in two calls of one step, on a stream that is not the current one at the time of the backward pass."""
    from crosslayer_transcoder_amd import custom_ops8 as C
    x, W = rnd(70, 2, 128, seed=1, spread=False).requires_grad_(), rnd(2, 128, 128, seed=2, spread=False).requires_grad_()
    want = [2 * g for g in torch.autograd.grad(C.plt_decoder8(x, W, None).sum(), (x, W))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss = C.plt_decoder8(x, W, None).sum() + C.plt_decoder8(x, W, None).sum()
    torch.cuda.current_stream().wait_stream(s)
    got = torch.autograd.grad(loss, (x, W))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))


@gpu
@pytest.mark.parametrize("dec", ["clt", "plt"])
def test_exported_and_compiled_models(dec):
    """torch.export of the whole model and torch.compile with batches of changing size, forward and every gradient, to the bit."""
    import crosslayer_transcoder_amd as cta
    from crosslayer_transcoder_amd.model import CrosslayerDecoder, CrossLayerTranscoder, Decoder, Encoder, ReLU
    torch.manual_seed(0)
    m = CrossLayerTranscoder(ReLU(), Encoder(96, 256, 2), (CrosslayerDecoder if dec == "clt" else Decoder)(96, 256, 2)).cuda()
    with cta.contractions8():
        x = rnd(20, 2, 96, seed=1, spread=False)
        with torch.no_grad():
            assert torch.equal(torch.export.export(m, (x,)).module()(x)[2], m(x)[2])
        c = torch.compile(m, backend="aot_eager", dynamic=True)
        for B in (20, 33, 7, 130):
            x, g = rnd(B, 2, 96, seed=B, spread=False).requires_grad_(), rnd(B, 2, 96, seed=B + 1, spread=False)
            leaves = [x] + list(m.parameters())
            y, z = c(x)[2], m(x)[2]
            assert torch.equal(y, z)
            assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y, leaves, g), torch.autograd.grad(z, leaves, g)))


@gpu
def test_checkpointed_offloaded_and_wrapped_tensors():
    """Recomputation, saved tensors on the host, a tensor class of its own, inference mode: the bits of a plain call."""
    from torch.utils.checkpoint import checkpoint
    from crosslayer_transcoder_amd import custom_ops8 as C

    class Wrapped(torch.Tensor):
        pass

    x, W, b = rnd(20, 2, 96, seed=1, spread=False), rnd(2, 96, 64, seed=2, spread=False).requires_grad_(), rnd(2, 64, seed=3, spread=False)
    want = C.plt_decoder8(x, W, b)
    dW, = torch.autograd.grad(want.sum(), W)
    assert torch.equal(torch.autograd.grad(checkpoint(lambda x: C.plt_decoder8(x, W, b), x, use_reentrant=False).sum(), W)[0], dW)
    with torch.autograd.graph.save_on_cpu():
        y = C.plt_decoder8(x, W, b)
    assert torch.equal(torch.autograd.grad(y.sum(), W)[0], dW)
    assert torch.equal(C.plt_decoder8(x.as_subclass(Wrapped), W, b).as_subclass(torch.Tensor), want)
    with torch.inference_mode():
        assert torch.equal(C.plt_decoder8(x, W, b), want)


def test_more_threads_than_a_launch_counts_are_refused():
    """Grids of more than 2^32 threads: errors before any launch (fewer blocks than 2^31, the count alone)."""
    from crosslayer_transcoder_amd._lib import lib
    p = 4096                                                                     # an aligned address nothing reads
    rows = 1 << 27
    assert lib.clt_unpack8(p, p, 0, 1, rows, 4096, 4096, rows, 0, 0, p, 1, None) == -6
    assert lib.clt_pack8(p, 1, 4096, 0, 1, rows, 4096, 0, 0, p, p, None, None, None, None, 0, None) == -6
    # results 2^23 elements apart, where only small tiles run: 2^13 x 2^13 of them
    n = 1 << 20
    assert lib.clt_gemm8(p, p, 0, 128, n, 0, 0, p, p, 0, 128, n, 0, 0, p, 1, 1 << 23, 0, None, 0, n, n, 128, 1, 0, None, 0, None) == -6
