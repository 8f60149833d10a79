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
