"""Performance cases of the operators behind a decoder: what turns its last hidden states into scores of tokens.

Four operators on device tensors, reached through ``excalibur_b200.capi`` (the C ABI), each reading what the one before
it writes:

* ``norm``: a block's result joins the residual stream (norm after the block, gate, residual scale) and the next block's
  norm is taken of the sum, in the activations' type or in 8-bit floating point with a scale for each 128 channels;
* ``quantize``: activations (a scale for each 128 channels of a row) or weights (for each 128 x 128) in 8-bit floating point;
* ``matmul``: the product of two such matrices;
* ``logprobs``: log probabilities of given tokens, the entropy and the most probable tokens of rows of logits.

``listed()`` are the fixed cases, ``draw(rng)`` gives others of the same ranges.
"""
import functools
import math

import torch

own = False      # False: the plain form below; True: the framework's kernels

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 128                    # channels that share a scale
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126   # of a block of zeros too: the scale's reciprocal stays finite


def listed():
    return [
        # one token of a decode step: the block's result joins the stream, the next norm is taken; latency counts
        _norm("norm_b1", 1, 4096, "f16", "rms", False, "none", False),
        # a prompt behind a block with a norm of its own and a gate by channel; the next product takes 8 bits
        _norm("norm_prompt_quantized", 4096, 4096, "bf16", "rms", True, "channel", True),
        # layer norm of an odd width, every sequence of 197 rows (a 14 x 14 map and one more) under a gate of its own
        _norm("norm_layer_odd", 3152, 1000, "f16", "layer", False, "group", False, group=197),
        # a decode batch's activations
        _quantize("quantize_b64", 64, 4096, "f16", 1),
        # the activations of a long prompt between the two products of a feed-forward block
        _quantize("quantize_prompt", 8192, 14336, "bf16", 1),
        # one token through a square projection: the weights are what is read
        _matmul("matmul_b1", 1, 4096, 4096, "f16", False),
        # a decode batch through a wide projection
        _matmul("matmul_b64_wide", 64, 14336, 4096, "bf16", False),
        # a classifier behind features of an odd width, a few hundred rows, with a bias
        _matmul("matmul_classes_odd", 333, 1000, 1234, "f16", True),
        # a long prompt through a large projection: arithmetic is what it costs
        _matmul("matmul_prompt", 8192, 8192, 8192, "f16", False),
        # one sampled token: its log probability and 20 alternatives, among as many tokens as large vocabularies have
        _logprobs("logprobs_b1", 1, 131072, "f32", 1, 20, 0.0),
        # scores of a prompt's own tokens, an odd vocabulary (rows at every alignment), a tenth of it masked
        _logprobs("logprobs_prompt_odd", 2048, 50001, "f16", 1, 5, 0.1),
        # the classifier's answers of a batch of images: 1000 classes, the five best
        _logprobs("logprobs_classes", 256, 1000, "f16", 1, 5, 0.0),
    ]


def _norm(name, rows, channels, dtype, kind, post, gate, quantized, group=1):
    return dict(name=name, op="norm", rows=rows, channels=channels, dtype=dtype, kind=kind, post=post, gate=gate, group=group,
                quantized=quantized)


def _quantize(name, rows, channels, dtype, block_rows):
    return dict(name=name, op="quantize", rows=rows, channels=channels, dtype=dtype, block_rows=block_rows)


def _matmul(name, m, n, k, out, bias):
    return dict(name=name, op="matmul", m=m, n=n, k=k, out=out, bias=bias)


def _logprobs(name, rows, vocab, dtype, given, top, masked):
    return dict(name=name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, given=given, top=top, masked=masked)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Widths of models: half of them whole multiples of 128, the others as they come."""
    w = _log(rng, lo, hi)
    return max(128, w // 128 * 128) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(("norm", "quantize", "matmul", "matmul", "logprobs"))
    if op == "norm":
        channels = _width(rng, 256, 16384)
        rows = _log(rng, 1, max(1, 4096 * 4096 // channels))
        gate = rng.choice(("none", "channel", "group", "row"))
        return {k: v for k, v in _norm("", rows, channels, rng.choice(("f16", "bf16", "f32") if rows * channels < 1 << 22 else ("f16", "bf16")),
                                       rng.choice(("rms", "rms", "layer")), rng.random() < 0.5, gate, rng.random() < 0.5,
                                       group=rng.randint(2, max(2, rows)) if gate == "group" else 1).items() if k != "name"}
    if op == "quantize":
        channels = _width(rng, 256, 16384)
        rows = _log(rng, 1, 8192 * 14336 // channels // 2)
        return {k: v for k, v in _quantize("", rows, channels, rng.choice(("f16", "bf16", "f32")), rng.choice((1, 1, 128))).items() if k != "name"}
    if op == "matmul":
        m, n, k = _log(rng, 1, 8192), _width(rng, 256, 16384), _width(rng, 256, 16384)
        m = min(m, 8192 ** 3 // (n * k))
        return {k_: v for k_, v in _matmul("", m, n, k, rng.choice(("f16", "bf16", "f32")), rng.random() < 0.3).items() if k_ != "name"}
    vocab = _log(rng, 1000, 262144)
    rows = _log(rng, 1, max(1, 2048 * 50001 // 2 // vocab))
    return {k: v for k, v in _logprobs("", rows, vocab, rng.choice(("f16", "bf16", "f32")), rng.choice((1, 1, 4)), rng.choice((0, 1, 5, 20)),
                                       rng.choice((0.0, 0.0, 0.5))).items() if k != "name"}


# ---- the plain forms: the operators as they are written down, in 32 bits ------------------------------------------------

def _normed(v, kind, weight, bias, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def _blocks(x, block_rows):
    """(rows, channels) in blocks of block_rows x 128, filled up with zeros: (row blocks, block_rows, channel blocks, 128)."""
    rows, channels = x.shape
    nr, nc = -(-rows // block_rows), -(-channels // BLOCK)
    x = torch.nn.functional.pad(x, (0, nc * BLOCK - channels, 0, nr * block_rows - rows))
    return x.reshape(nr, block_rows, nc, BLOCK)


def _quantized(x, block_rows):
    """e4m3 values (rows, channels), and scales: (channel blocks, rows) of single rows, (row blocks, channel blocks) otherwise."""
    rows, channels = x.shape
    b = _blocks(x, block_rows)
    scales = (b.abs().amax((1, 3), keepdim=True) / E4M3_MAX).clamp_min(SMALLEST_SCALE)
    q = (b * (1.0 / scales)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    q = q.reshape(q.shape[0] * block_rows, -1)[:rows, :channels]
    scales = scales[:, 0, :, 0]
    return q, scales.t().contiguous() if block_rows == 1 else scales.contiguous()


def _plain_norm(s):
    v = s["h"].float()
    if s["post"] is not None:
        v = _normed(v, s["kind"], s["post"], s["post_bias"], s["eps"])
    if s["gate"] is not None:
        v = v * (s["gate"].float().repeat_interleave(s["group"], 0)[:v.shape[0]] if s["group"] else s["gate"].float())
    v = s["x"].float() + s["residual_scale"] * v
    n = _normed(v, s["kind"], s["weight"], s["bias"], s["eps"])
    r = v.to(s["h"].dtype)
    return (r, *_quantized(n, 1)) if s["quantized"] else (r, n.to(s["h"].dtype))


def _dequantized(q, scales, block_rows):
    """The values that e4m3 matrices with their scales stand for."""
    if block_rows == 1:
        return q.float() * scales.t().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
    return q.float() * scales.repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _plain_matmul(s):
    y = _dequantized(s["a"], s["a_scales"], 1) @ _dequantized(s["w"], s["w_scales"], BLOCK).t()
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"])


def _best(z, top):
    """The indexes of the `top` largest of every row, equal ones by their index: keys of value and index are all different."""
    bits = (z + 0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32) - torch.arange(z.shape[1], device=z.device)
    return keys.topk(top, -1, sorted=True).indices


def _plain_logprobs(s):
    z = s["logits"].float() * s["scale"]
    m = z.amax(-1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(-1, keepdim=True)
    lp = z - m - total.log()
    given = lp.gather(1, s["tokens"].long())
    entropy = -(torch.where(e > 0, lp, 0.0) * e / total).sum(-1)
    if not s["top"]:
        return given, entropy
    best = _best(s["logits"].float(), s["top"])
    return given, entropy, lp.gather(1, best), best.int()


# ---- the framework's calls ----------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _context():
    from excalibur_b200 import capi
    return capi, capi.Context(torch.cuda.current_device())


def _own_norm(s):
    capi, ctx = _context()
    return capi.residual_norm(ctx, s["h"], s["x"], post_weight=s["post"], post_bias=s["post_bias"], gate=s["gate"], gate_rows=s["group"],
                              residual_scale=s["residual_scale"], weight=s["weight"], bias=s["bias"],
                              kind=capi.NORM_LAYER if s["kind"] == "layer" else capi.NORM_RMS, eps=s["eps"], quantized=s["quantized"])


def _own_quantize(s):
    capi, ctx = _context()
    return capi.quantize_blocks(ctx, s["x"], block_rows=s["block_rows"])


def _own_matmul(s):
    capi, ctx = _context()
    return capi.fp8_matmul(ctx, s["a"], s["a_scales"], s["w"], s["w_scales"], bias=s["bias"], out_dtype=capi.exb_dtype_of(s["out"]))


def _own_logprobs(s):
    capi, ctx = _context()
    got = capi.token_logprobs(ctx, s["logits"], s["tokens"], top=s["top"], scale=s["scale"])
    return got if s["top"] else got[:2]


def _plain_quantize(s):
    return _quantized(s["x"].float(), s["block_rows"])


def run(state):
    op = state["op"]
    if own:
        return {"norm": _own_norm, "quantize": _own_quantize, "matmul": _own_matmul, "logprobs": _own_logprobs}[op](state)
    return {"norm": _plain_norm, "quantize": _plain_quantize, "matmul": _plain_matmul, "logprobs": _plain_logprobs}[op](state)


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _activations(gen, rows, channels, dtype):
    """Hidden states: normal values, and a few channels that are much larger, as trained models have them."""
    x = torch.randn((rows, channels), device="cuda", generator=gen)
    loud = torch.rand(channels, device="cuda", generator=gen) < 0.004
    return x.mul_(torch.where(loud, 20.0, 1.0)).to(dtype)


def _rows_of_16(q):
    """The same matrix with rows that start at multiples of 16 bytes, as the quantiser writes them."""
    rows, channels = q.shape
    wide = torch.zeros((rows, (channels + 15) // 16 * 16), device=q.device, dtype=torch.uint8)
    wide[:, :channels] = q.view(torch.uint8)
    return wide.view(torch.float8_e4m3fn)[:, :channels]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = functools.partial(torch.randn, device="cuda", generator=gen)
    op = case["op"]
    if op == "norm":
        rows, channels, dtype = case["rows"], case["channels"], DTYPES[case["dtype"]]
        layer = case["kind"] == "layer"
        group = {"none": 0, "channel": 0, "group": case["group"], "row": 1}[case["gate"]]
        gates = {"none": 0, "channel": 1, "group": -(-rows // case["group"]), "row": rows}[case["gate"]]
        return dict(op=op, kind=case["kind"], quantized=case["quantized"], group=group, eps=1e-5, residual_scale=0.22,
                    h=_activations(gen, rows, channels, dtype), x=_activations(gen, rows, channels, dtype),
                    post=1 + 0.1 * rand(channels) if case["post"] else None,
                    post_bias=0.1 * rand(channels) if case["post"] and layer else None,
                    gate=torch.tanh(rand(gates, channels)).to(dtype) if gates else None,
                    weight=1 + 0.1 * rand(channels), bias=0.1 * rand(channels) if layer else None)
    if op == "quantize":
        return dict(op=op, x=_activations(gen, case["rows"], case["channels"], DTYPES[case["dtype"]]), block_rows=case["block_rows"])
    if op == "matmul":
        a, a_scales = _quantized(_activations(gen, case["m"], case["k"], torch.float32), 1)
        w, w_scales = _quantized(rand(case["n"], case["k"]).mul_(0.02), BLOCK)
        return dict(op=op, a=_rows_of_16(a), a_scales=a_scales, w=_rows_of_16(w), w_scales=w_scales, out=DTYPES[case["out"]],
                    bias=rand(case["n"]) if case["bias"] else None)
    rows, vocab = case["rows"], case["vocab"]
    logits = rand(rows, vocab).mul_(2.5)
    tokens = torch.randint(0, vocab, (rows, case["given"]), device="cuda", generator=gen)
    if case["masked"]:
        logits.masked_fill_(torch.rand((rows, vocab), device="cuda", generator=gen) < case["masked"], -math.inf)
        logits.scatter_(1, tokens, rand(rows, case["given"]))         # what is asked for is among what is left
    logits.scatter_add_(1, tokens[:, :1], 6 * torch.rand((rows, 1), device="cuda", generator=gen))      # and more probable than most
    return dict(op=op, logits=logits.to(DTYPES[case["dtype"]]), tokens=tokens.int(), top=case["top"], scale=1.25)


def work(case):
    op = case["op"]
    if op == "norm":
        n, es = case["rows"] * case["channels"], SIZES[case["dtype"]]
        gates = {"none": 0, "channel": 1, "group": -(-case["rows"] // case["group"]), "row": case["rows"]}[case["gate"]]
        out = 1 + 4 / BLOCK if case["quantized"] else es
        return {"bytes": n * (3 * es + out) + (gates * es + 8) * case["channels"], "flops": n * (14 if case["post"] else 9)}
    if op == "quantize":
        n = case["rows"] * case["channels"]
        return {"bytes": n * (SIZES[case["dtype"]] + 1) + 4 * n / BLOCK / case["block_rows"], "flops": 3 * n}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + m * n * SIZES[case["out"]] + 4 * m * k / BLOCK + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * SIZES[case["dtype"]] + case["rows"] * (8 * case["given"] + 8 * case["top"] + 4), "flops": 6 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _to_e4m3(v):
    """The nearest of the numbers with 4 significant bits, whole multiples of 2^-9 and at most 448; ties to the even one."""
    exponent = torch.frexp(v).exponent.clamp_min(-5)
    step = torch.ldexp(torch.ones_like(v), exponent - 4)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quantized(x, block_rows):
    rows, channels = x.shape
    nr, nc = -(-rows // block_rows), -(-channels // 128)
    wide = x.new_zeros((nr * block_rows, nc * 128))
    wide[:rows, :channels] = x
    largest = wide.abs().view(nr, block_rows, nc, 128).amax(3).amax(1)
    scales = torch.maximum(largest / E4M3_MAX, largest.new_tensor(SMALLEST_SCALE))
    each = scales.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)
    return _to_e4m3((wide / each)[:rows, :channels]), scales.t() if block_rows == 1 else scales


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        return _exact_quantized(s["x"].double(), s["block_rows"])
    if s["op"] == "matmul":
        a, w = s["a"].double(), s["w"].double()
        for k in range(0, a.shape[1], 128):
            b = k // 128
            a[:, k:k + 128] *= s["a_scales"][b].double()[:, None]
            w[:, k:k + 128] *= s["w_scales"][:, b].double().repeat_interleave(128)[:w.shape[0], None]
        y = torch.einsum("mk,nk->mn", a, w)
        return y if s["bias"] is None else y + s["bias"].double()
    if s["op"] == "norm":
        def norm(v, weight, bias):
            mean = v.mean(1, keepdim=True) if s["kind"] == "layer" else 0.0
            spread = ((v - mean) ** 2).mean(1, keepdim=True) + s["eps"]
            return (v - mean) / spread.sqrt() * weight.double() + (0.0 if bias is None else bias.double())
        v = s["h"].double()
        if s["post"] is not None:
            v = norm(v, s["post"], s["post_bias"])
        if s["gate"] is not None:
            at = torch.arange(v.shape[0], device=v.device) // s["group"] if s["group"] else torch.zeros(v.shape[0], device=v.device, dtype=torch.long)
            v = v * s["gate"].double()[at]
        r = s["x"].double() + s["residual_scale"] * v
        n = norm(r, s["weight"], s["bias"])
        return (r, *_exact_quantized(n, 1)) if s["quantized"] else (r, n)
    z = s["logits"].double() * s["scale"]
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = (z - lse).exp()
    entropy = lse[:, 0] - torch.where(p > 0, p * z, 0.0).sum(1)
    given = z.gather(1, s["tokens"].long()) - lse
    if not s["top"]:
        return given, entropy
    values, order = z.sort(dim=1, descending=True, stable=True)
    return given, entropy, values[:, :s["top"]] - lse, order[:, :s["top"]].int()
