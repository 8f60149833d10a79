"""The 8-bit block-scaled operators at the sizes they are used at: activation checkpoints in 8 bits, products of 8-bit
matrices with kept weights, and the training step of a linear map that keeps its input in 8 bits for the backward pass.

A matrix [R, C] is held in 8-bit floats (e4m3: 4 exponent and 3 mantissa bits, largest 448; e5m2: 5 and 2, largest 57344)
with one scale 2^e for every row and block of 128 columns.  e is the smallest integer >= -112 with
max |x| <= largest * 2^e over the block; the code is x * 2^-e rounded to nearest, ties to even.  Blocks of a weight matrix
are 128 x 128, so that its transposed copy holds the same values.  The products are those of the values so held."""
import math

import torch

own = False

BLOCK = 128
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}

# op "checkpoint": x [T, L, K] is packed and restored; form "rows" holds it in blocks along K, "columns" in blocks of 128 tokens
#   (transposed: what a weight gradient contracts over), "both" makes the two in one call.
# op "product":    y [T, L, N] = x [T, L, K] (packed in the call) times weights that a program keeps in 8 bits, plus a bias.
# op "train":      y = x W + b and its gradients for a given dy; side "encoder" keeps W as [L, N, K] in memory, "decoder" as
#   [L, K, N].  y and dx have x's type, dW and db are float32 like the parameters.


def listed():
    return [
        # the debug configuration's batch (config/debug-cpu.yaml: 2 layers of 110 values, 16 tokens): latency alone
        {"name": "checkpoint_debug", "op": "checkpoint", "T": 16, "L": 2, "K": 110, "x": "float32", "fmt": "e4m3", "form": "both"},
        # odd sizes in every direction, the wide-range format, fp16 activations
        {"name": "checkpoint_ragged", "op": "checkpoint", "T": 1000, "L": 3, "K": 2049, "x": "float16", "fmt": "e5m2", "form": "columns"},
        # features of four layers of a 32k dictionary for a training batch of 4096 tokens
        {"name": "checkpoint_features", "op": "checkpoint", "T": 4096, "L": 4, "K": 32768, "x": "bfloat16", "fmt": "e4m3", "form": "both"},
        # features of one layer for the token being generated: one pass over the weights
        {"name": "one_token_encoder", "op": "product", "T": 1, "L": 1, "K": 768, "N": 32768, "x": "bfloat16", "y": "bfloat16"},
        # reconstruction of the last layer from the features of all 12 layers, one token: a long contraction
        {"name": "one_token_decoder", "op": "product", "T": 1, "L": 1, "K": 393216, "N": 768, "x": "bfloat16", "y": "float32"},
        # features of every layer for a batch of 32 requests
        {"name": "requests_all_layers", "op": "product", "T": 32, "L": 12, "K": 768, "N": 32768, "x": "bfloat16", "y": "bfloat16"},
        # the encoder of the 12-layer 32k transcoder on a whole batch
        {"name": "batch_all_layers", "op": "product", "T": 4096, "L": 12, "K": 768, "N": 32768, "x": "bfloat16", "y": "bfloat16"},
        # odd sizes, 32-bit activations and results
        {"name": "batch_ragged", "op": "product", "T": 1000, "L": 3, "K": 2049, "N": 5003, "x": "float32", "y": "float32"},
        # a training step of the debug configuration's encoder
        {"name": "train_debug", "op": "train", "side": "encoder", "T": 16, "L": 2, "K": 110, "N": 32, "x": "float32", "dx": True},
        # the encoder of the 12-layer transcoder: the activations are data, no gradient leaves through them
        {"name": "train_encoder", "op": "train", "side": "encoder", "T": 4096, "L": 12, "K": 768, "N": 32768, "x": "bfloat16", "dx": False},
        # a per-layer decoder with 8k features a layer
        {"name": "train_decoder", "op": "train", "side": "decoder", "T": 4096, "L": 12, "K": 8192, "N": 768, "x": "bfloat16", "dx": True},
        # one layer of a transcoder for a model of width 4096
        {"name": "train_wide", "op": "train", "side": "encoder", "T": 2048, "L": 1, "K": 4096, "N": 32768, "x": "bfloat16", "dx": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["checkpoint", "product", "train"])
    while True:
        c = {"op": op, "T": _log(rng, 1, 4096), "L": _log(rng, 1, 12), "K": _log(rng, 16, 32768),
             "x": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
        if op == "checkpoint":
            c |= {"fmt": rng.choice(["e4m3", "e5m2"]), "form": rng.choice(["rows", "columns", "both"])}
        else:
            c["N"] = _log(rng, 16, 32768)
            if op == "product":
                c["y"] = rng.choice(["bfloat16", "float16", "float32"])
            else:
                c |= {"side": rng.choice(["encoder", "decoder"]), "dx": rng.random() < 0.7}
            if rng.random() < 0.5:          # model widths and dictionaries are mostly multiples of 64
                c["K"], c["N"] = max(64, c["K"] // 64 * 64), max(64, c["N"] // 64 * 64)
        w = work(c)
        if w["bytes"] <= 6e9 and w["flops"] <= 2.4e12 and c["L"] * c.get("N", 0) * c["K"] <= 3.0e8:
            return c


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _up(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, L, K, dt = case["T"], case["L"], case["K"], DT[case["x"]]
    s = dict(case)
    if case["op"] == "checkpoint" or case.get("side") == "decoder" or K > 8192:
        x = torch.relu(_randn(g, T, L, K) - 1.0)                    # features: positive, most of them zero
    else:
        x = _randn(g, T, L, K) * (0.5 + torch.rand((L, K), generator=g, device="cuda"))
    x[:1] *= 20.0                                                   # a first token is far larger than the others
    s["x"] = x.to(dt)
    del x
    if case["op"] == "checkpoint":
        return s
    N = case["N"]
    s["b"] = _randn(g, L, N) * 0.05
    if case["op"] == "product":
        # weights as a program keeps them: codes [L, N, K rounded up to 128] (zero behind K), scale bytes e + 127
        # [L, K blocks, N rounded up to 128]
        kb, codes = _up(K) // BLOCK, torch.empty(0)
        codes = (torch.rand((L, N, _up(K)), generator=g, device="cuda") * 800.0 - 400.0).to(F8["e4m3"]).view(torch.uint8)
        codes[:, :, K:] = 0
        e = torch.randint(-16, -11, (L, kb, _up(N) // BLOCK), generator=g, device="cuda")
        s["codes"], s["scale"] = codes, (e + 127).to(torch.uint8).repeat_interleave(BLOCK, dim=2).contiguous()
        s["y_type"] = DT[case["y"]]
        return s
    bound = 1.0 / math.sqrt(max(N, K))
    shape = (L, N, K) if case["side"] == "encoder" else (L, K, N)
    s["W"] = (torch.rand(shape, generator=g, device="cuda") * 2 - 1) * bound
    if case["side"] == "encoder":
        s["W"] = s["W"].permute(0, 2, 1)                            # [L, K, N], feature-major in memory
    s["dy"] = (_randn(g, T, L, N) * 1e-3).to(dt)
    return s


# ---- plain form ---------------------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e, -126 <= e <= 127, put together from its bits: exp2 and ldexp may be off by a rounding, which moves ties."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _held(x, fmt, rows=1):
    """Values that x [..., R, C] has when held in 8 bits with a scale for every `rows` rows and 128 columns."""
    R, C = x.shape[-2:]
    x = torch.nn.functional.pad(x.float(), (0, -C % BLOCK, 0, -R % rows))
    v = x.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, rows))                    # [..., R / rows, rows, C / 128, 128]
    m, p = torch.frexp(v.abs().amax(dim=(-1, -3), keepdim=True))                  # max = m * 2^p, 0.5 <= m < 1; largest = 0.875 * 2^q
    q = 9 if fmt == "e4m3" else 16
    e = (p - q + (m > 0.875)).clamp(min=-112)
    v = (v * _pow2(-e)).to(F8[fmt]).float() * _pow2(e)
    return v.flatten(-2).flatten(-3, -2)[..., :R, :C]


def _train_plain(x, W, b, dy, need_dx):
    dt, x, dy = x.dtype, x.transpose(0, 1), dy.transpose(0, 1)                    # [L, T, .]
    w = _held(W, "e4m3", rows=BLOCK)                                              # [L, K, N]
    y = torch.matmul(_held(x, "e4m3"), w) + b[:, None]
    xt, dyt = _held(x.mT, "e4m3"), _held(dy.mT, "e4m3")                           # blocks of 128 tokens
    dW = torch.matmul(xt, dyt.mT)
    dx = torch.matmul(_held(dy, "e4m3"), w.mT).transpose(0, 1).to(dt) if need_dx else None
    return [y.transpose(0, 1).to(dt), dx, dW, dy.float().sum(1)]


def run(s):
    x = s["x"]
    if s["op"] == "checkpoint":
        v = x.transpose(0, 1)                                                     # [L, T, K]
        if own:
            from crosslayer_transcoder_amd import ops8
            if s["form"] == "both":
                q, qt = ops8.quantize8_both(v, s["fmt"])
                return [ops8.dequantize8(q, x.dtype), ops8.dequantize8(qt, x.dtype)]
            return [ops8.dequantize8((ops8.quantize8 if s["form"] == "rows" else ops8.quantize8_t)(v, s["fmt"]), x.dtype)]
        out = [_held(v, s["fmt"])] if s["form"] != "columns" else []
        return [o.to(x.dtype) for o in out + ([_held(v.mT, s["fmt"])] if s["form"] != "rows" else [])]
    if s["op"] == "product":
        if own:
            from crosslayer_transcoder_amd import ops8
            w = ops8.Block8(s["codes"], s["scale"], s["N"], s["K"], "e4m3")
            return ops8.linear8(x, w, s["b"], out_dtype=s["y_type"])
        scale = _pow2(s["scale"].to(torch.int32) - 127).mT[:, :s["N"], :, None]     # [L, N, K blocks, 1]
        w = (s["codes"].view(F8["e4m3"]).float().unflatten(-1, (-1, BLOCK)) * scale).flatten(-2)[..., :s["K"]]
        y = torch.matmul(_held(x.transpose(0, 1), "e4m3"), w.mT) + s["b"][:, None]
        return y.transpose(0, 1).to(s["y_type"])
    if own:
        from crosslayer_transcoder_amd import custom_ops8
        x, W, b = x.detach().requires_grad_(s["dx"]), s["W"].detach().requires_grad_(), s["b"].detach().requires_grad_()
        y = (custom_ops8.encoder8 if s["side"] == "encoder" else custom_ops8.plt_decoder8)(x, W, b)
        grads = torch.autograd.grad(y, ([x] if s["dx"] else []) + [W, b], s["dy"])
        return [y.detach(), grads[0] if s["dx"] else None, grads[-2], grads[-1]]
    return _train_plain(x, s["W"], s["b"], s["dy"], s["dx"])


# ---- work: what the operator reads and writes once, and its products ------------------------------------------------------
def work(case):
    T, L, K = case["T"], case["L"], case["K"]
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    ex = size[case["x"]]
    if case["op"] == "checkpoint":
        n, forms = T * L * K, 2 if case["form"] == "both" else 1
        return {"bytes": n * ex + forms * n * (2 * (1 + 1 / BLOCK) + ex), "flops": 4 * n * forms}     # x; codes written and read; restored
    N = case["N"]
    if case["op"] == "product":
        return {"bytes": L * (N * K * (1 + 1 / BLOCK) + T * K * ex + T * N * size[case["y"]] + 4 * N), "flops": 2 * L * T * N * K}
    products = 3 if case["dx"] else 2
    # forward: x, W in, y out, x kept in 8 bits (and W, for dx); backward: dy and what was kept in, dx, dW, db out
    by = T * K * ex + 4 * N * K + T * N * ex + 2 * T * K + T * N * ex + 4 * N * K + 8 * N
    by += (T * K * ex + 2 * N * K) if case["dx"] else 0
    return {"bytes": L * by, "flops": 2 * products * L * T * N * K}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_held(x, fmt, tiles=False):
    """x [L, R, C] in float64, block by block from the definition: the exponent by comparison, the code by rounding to the
    format's step at its magnitude."""
    L, R, C = x.shape
    r, low, bits = (BLOCK if tiles else 1), (-6 if fmt == "e4m3" else -14), (3 if fmt == "e4m3" else 2)
    big = torch.zeros((L, -(-R // r) * r, _up(C)), dtype=torch.float64, device=x.device)
    big[:, :R, :C] = x.double().abs()
    top = big.view(L, -1, r, _up(C) // BLOCK, BLOCK).amax(4).amax(2)              # [L, R / r, C / 128]
    del big
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / LARGEST[fmt])) - 1
    for _ in range(3):
        e = torch.where(top > LARGEST[fmt] * _two_to(e), e + 1, e)
    scale = _two_to(e.clamp(min=-112.0)).repeat_interleave(r, 1)[:, :R].repeat_interleave(BLOCK, 2)[:, :, :C]
    v = x.double() / scale
    p = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40)))
    p = torch.where(v.abs() < _two_to(p), p - 1, p)
    p = torch.where(v.abs() >= _two_to(p + 1), p + 1, p)
    step = _two_to(p.clamp(min=low) - bits)
    return torch.round(v / step) * step * scale


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].transpose(0, 1)
    if case["op"] == "checkpoint":
        out = [_exact_held(x, case["fmt"])] if case["form"] != "columns" else []
        return out + ([_exact_held(x.transpose(1, 2), case["fmt"])] if case["form"] != "rows" else [])
    if case["op"] == "product":
        w = s["codes"].view(F8["e4m3"]).double()[:, :, :case["K"]]
        e = (s["scale"].double() - 127).transpose(1, 2).repeat_interleave(BLOCK, 2)[:, :case["N"], :case["K"]]
        w = w * _two_to(e)
        del e
        y = torch.bmm(_exact_held(x, "e4m3"), w.transpose(1, 2).contiguous())
        return (y + s["b"].double()[:, None]).transpose(0, 1).contiguous()
    W = _exact_held(s["W"], "e4m3", tiles=True)
    dy = s["dy"].transpose(0, 1)
    y = (torch.bmm(_exact_held(x, "e4m3"), W) + s["b"].double()[:, None]).transpose(0, 1).contiguous()
    dx = None
    if case["dx"]:
        dx = torch.bmm(_exact_held(dy, "e4m3"), W.transpose(1, 2).contiguous()).transpose(0, 1).contiguous()
    del W
    xt, dyt = _exact_held(x.transpose(1, 2), "e4m3"), _exact_held(dy.transpose(1, 2), "e4m3")
    dW = torch.bmm(xt, dyt.transpose(1, 2).contiguous())
    return [y, dx, dW, dy.double().sum(1)]
