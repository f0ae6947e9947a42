"""Performance cases of the operators of decoding in 8-bit integers, by experts and with beams.

Operators on device tensors, reached through ``excalibur_b200.capi`` (the C ABI):

* ``linear``: activations to 8-bit integers with a scale for each row (``quantize_rows``), times weights in 8-bit integers with a
  scale for each output channel (``int8_matmul``);
* ``experts``: rows sorted by expert, each times its expert's weights (``grouped_matmul``): in 8-bit integers behind ``quantize_rows``,
  in fp16 or bf16;
* ``beams``: the best continuations of every sentence over its beams and the vocabulary (``beam_select``);
* ``reorder``: the beams' states follow their parents, in place (``reorder_beams``).

``listed()`` are the fixed cases, ``draw(rng)`` gives others of the same ranges.
"""
import functools
import math

import torch

own = False      # False: the plain form below; True: the framework's kernels

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"int8": 1, "f16": 2, "bf16": 2, "f32": 4}
SMALLEST_SCALE = 2.0 ** -126   # of a row of zeros too: the scale's reciprocal stays finite


def listed():
    return [
        # one token of a decode step through a square projection: the weights are what is read, latency counts
        _linear("linear_b1", 1, 4096, 4096, "f16", False),
        # a decode batch through a wide projection
        _linear("linear_b64_wide", 64, 14336, 4096, "bf16", False),
        # a classifier behind features of an odd width, a few hundred rows, with a bias
        _linear("linear_classes_odd", 333, 1000, 1234, "f16", True),
        # a long prompt through a large projection: arithmetic is what it costs
        _linear("linear_prompt", 8192, 8192, 8192, "f16", False),
        # one token that goes to two of eight experts
        _experts("experts_b1", 2, 4096, 4096, "f16", 8, 2, False),
        # a decode batch over many small experts of odd sizes, some without a row
        _experts("experts_batch_odd", 509, 1500, 2000, "int8", 64, 61, True),
        # a prompt, two of eight large experts a token
        _experts("experts_prompt", 8192, 14336, 4096, "bf16", 8, 8, False),
        # one sentence, four beams, as many tokens as large vocabularies have
        _beams("beams_b1", 1, 4, 131072, "f32", 8, 0, 0.0),
        # a batch of sentences, an odd vocabulary (rows at every alignment), a tenth of it masked, some beams ended
        _beams("beams_batch_odd", 64, 5, 50001, "bf16", 10, 1, 0.1),
        # many sentences of a large vocabulary
        _beams("beams_many", 128, 8, 131072, "f16", 8, 0, 0.0),
        # the cache of one sentence: 32 layers' keys and values
        _reorder("reorder_b1", 1, 4, 64, 8, 1024, 128, "f16", 2),
        # the cache of a batch of sentences of unlike lengths: 8 layers' keys and values
        _reorder("reorder_batch", 16, 8, 16, 8, 2048, 64, "bf16", 6),
    ]


def _linear(name, m, n, k, dtype, bias):
    return dict(name=name, op="linear", m=m, n=n, k=k, dtype=dtype, bias=bias)


def _experts(name, m, n, k, dtype, experts, used, bias):
    return dict(name=name, op="experts", m=m, n=n, k=k, dtype=dtype, experts=experts, used=used, bias=bias)


def _beams(name, sentences, beams, vocab, dtype, select, ended, masked):
    return dict(name=name, op="beams", sentences=sentences, beams=beams, vocab=vocab, dtype=dtype, select=select, ended=ended, masked=masked)


def _reorder(name, sentences, beams, states, heads, positions, channels, dtype, moved):
    return dict(name=name, op="reorder", sentences=sentences, beams=beams, states=states, heads=heads, positions=positions, channels=channels, dtype=dtype,
                moved=moved)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi, step=1):
    """Widths of models: half of them whole multiples of 128, the others as they come (whole multiples of `step`)."""
    w = _log(rng, lo, hi)
    return max(128, w // 128 * 128) if rng.random() < 0.5 else max(step, w // step * step)


def draw(rng):
    op = rng.choice(("linear", "linear", "experts", "experts", "beams", "reorder"))
    if op == "linear":
        m, n, k = _log(rng, 1, 8192), _width(rng, 256, 16384), _width(rng, 256, 16384)
        case = _linear("", min(m, 8192 ** 3 // (n * k)), n, k, rng.choice(("f16", "bf16", "f32")), rng.random() < 0.3)
    elif op == "experts":
        dtype = rng.choice(("int8", "f16", "bf16"))
        n, k = _width(rng, 256, 8192), _width(rng, 256, 8192, 1 if dtype == "int8" else 8)
        experts = min(_log(rng, 2, 128), 8 * 14336 * 4096 // (n * k))
        m = min(_log(rng, 1, 8192), 8192 * 14336 * 4096 // (4 * n * k))
        most = min(m, experts)
        case = _experts("", m, n, k, dtype, experts, rng.randint((most + 1) // 2, most), rng.random() < 0.3)
    elif op == "beams":
        beams, vocab = rng.randint(1, 16), _log(rng, 1000, 262144)
        sentences = min(_log(rng, 1, 256), max(1, 128 * 8 * 131072 // (2 * beams * vocab)))
        case = _beams("", sentences, beams, vocab, rng.choice(("f16", "bf16", "f32")), rng.choice((beams, 2 * beams)), rng.randint(0, beams // 3),
                      rng.choice((0.0, 0.0, 0.5)))
    else:
        sentences, beams, heads, channels = _log(rng, 1, 32), rng.randint(2, 16), rng.randint(1, 32), rng.choice((64, 80, 96, 128, 256, rng.randint(16, 256)))
        dtype = rng.choice(("f16", "bf16", "f32"))
        row = heads * channels * SIZES[dtype]
        positions = min(_log(rng, 16, 8192), max(1, 128 * 8 * 2048 * 64 * 2 // (sentences * beams * row)))
        states = min(2 * _log(rng, 1, 30), max(1, 16 * 128 * 8 * 2048 * 64 * 2 // (sentences * beams * row * positions)))
        case = _reorder("", sentences, beams, states, heads, positions, channels, dtype, rng.randint(1, beams - 1))
    del case["name"]
    return case


# ---- the plain forms: the operators as they are written down, in 32 bits ------------------------------------------------

def _quantized(x):
    """Whole numbers from -127 to 127, as fp32, and each row's scale (a quotient of tensors: one of a tensor and a number is a product).
    The products are in 64 bits, where they are exact: in 32 some would fall on the other side of a border between two numbers."""
    largest = x.abs().amax(-1, keepdim=True)
    scales = (largest / torch.full_like(largest, 127.0)).clamp_min(SMALLEST_SCALE)
    return torch.round(x.double() * (1.0 / scales).double()).float(), scales


def _plain_linear(s):
    q, scales = _quantized(s["x"].float())
    y = (q @ s["w"].float().t()) * (scales * s["w_scales"])
    return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)


def _plain_experts(s):
    """The rows of each expert in a batch of their own, filled up to the longest."""
    x, ends = s["x"].float(), s["ends"].long()
    scales = s["w_scales"]
    if scales is not None:
        x, row_scales = _quantized(x)
    starts = torch.nn.functional.pad(ends[:-1], (1, 0))
    at = (starts[:, None] + torch.arange(s["longest"], device=x.device)).clamp_max(x.shape[0] - 1)
    each = torch.bmm(x[at], s["w"].float().transpose(1, 2))
    row = torch.arange(x.shape[0], device=x.device)
    expert = (row[:, None] >= ends).sum(1)
    y = each[expert, row - starts[expert]]
    if scales is not None:
        y = y * (row_scales * scales[expert])
    return (y if s["bias"] is None else y + s["bias"][expert]).to(s["x"].dtype)


def _best(z, top):
    """The indexes of the `top` largest of every row, equal ones by their index: keys of value and index are all different."""
    bits = (z + 0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32) - torch.arange(z.shape[1], device=z.device)
    return keys.topk(top, -1, sorted=True).indices


def _plain_beams(s):
    """In 64 bits: what is selected must not hang on the rounding of sums."""
    scores, select, vocab = s["scores"].double(), s["select"], s["logits"].shape[1]
    sentences, beams = scores.shape
    z = s["logits"].double() * s["scale"]
    m = z.amax(-1, keepdim=True)
    lse = m + (z - m).exp().sum(-1, keepdim=True).log()
    tokens = _best(s["logits"].float(), select)
    each = scores.reshape(-1, 1) + (z.gather(1, tokens) - lse)
    if s["ended"] is not None:      # an ended beam goes on with one token, at no cost
        first = torch.arange(select, device=z.device) == 0
        stay = torch.where(first, scores.reshape(-1, 1), -math.inf)
        ended = s["ended"].reshape(-1, 1)
        each, tokens = torch.where(ended, stay, each), torch.where(ended, s["end_token"], tokens)
    each, tokens = each.reshape(sentences, -1), tokens.reshape(sentences, -1)
    got, order = each.sort(dim=1, descending=True, stable=True)      # equal scores: the lower beam, then the order in it
    got, order = got[:, :select], order[:, :select]
    none = got == -math.inf
    return got.float(), torch.where(none, -1, order // select).int(), torch.where(none, -1, tokens.gather(1, order)).int()


def _plain_reorder(s):
    cache, parents, lengths = s["cache"], s["parents"].long(), s["lengths"]
    sentences, beams = parents.shape
    rows = (parents + torch.arange(sentences, device=cache.device)[:, None] * beams).reshape(-1)
    below = torch.arange(cache.shape[3], device=cache.device) < lengths.repeat_interleave(beams)[:, None]
    cache.copy_(torch.where(below[None, :, None, :, None], cache[:, rows], cache))
    return cache


# ---- the framework's calls ----------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _context():
    from excalibur_b200 import capi
    return capi, capi.Context(torch.cuda.current_device())


def _own_linear(s):
    capi, ctx = _context()
    q, scales = capi.quantize_rows(ctx, s["x"])
    return capi.int8_matmul(ctx, q, scales, s["w"], s["w_scales"], bias=s["bias"], out_dtype=capi.exb_dtype_of(s["x"]))


def _own_experts(s):
    capi, ctx = _context()
    x, scales = s["x"], None
    if s["w_scales"] is not None:
        x, scales = capi.quantize_rows(ctx, x)
    return capi.grouped_matmul(ctx, x, s["w"], s["ends"], a_scales=scales, w_scales=s["w_scales"], bias=s["bias"], out_dtype=capi.exb_dtype_of(s["x"]))


def _own_beams(s):
    capi, ctx = _context()
    return capi.beam_select(ctx, s["logits"], s["scores"], s["select"], scale=s["scale"], ended=s["ended"], end_token=s["end_token"])


def _own_reorder(s):
    capi, ctx = _context()
    capi.reorder_beams(ctx, s["layers"], s["parents"], lengths=s["lengths"])
    return s["cache"]


def run(state):
    op = state["op"]
    if own:
        return {"linear": _own_linear, "experts": _own_experts, "beams": _own_beams, "reorder": _own_reorder}[op](state)
    return {"linear": _plain_linear, "experts": _plain_experts, "beams": _plain_beams, "reorder": _plain_reorder}[op](state)


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _activations(gen, rows, channels, dtype):
    """Hidden states: normal values, and a few channels that are much larger, as trained models have them."""
    x = torch.randn((rows, channels), device="cuda", generator=gen)
    loud = torch.rand(channels, device="cuda", generator=gen) < 0.004
    return x.mul_(torch.where(loud, 20.0, 1.0)).to(dtype)


def _weights(rand, *shape):
    """8-bit integers in rows that start at multiples of 16 bytes, as quantize_rows writes them, and a scale for each row."""
    q, scales = _quantized(rand(*shape).mul_(0.02))
    wide = torch.zeros((*shape[:-1], (shape[-1] + 15) // 16 * 16), device=q.device, dtype=torch.int8)
    wide[..., :shape[-1]] = q
    return wide[..., :shape[-1]], scales[..., 0].contiguous()


def _ends(gen, rows, experts, used):
    """Rows of `used` of the experts, one at least each, some up to four times as likely as others: where each expert's rows end."""
    who = torch.randperm(experts, device="cuda", generator=gen)[:used]
    weight = 0.25 + 0.75 * torch.rand(used, device="cuda", generator=gen)
    more = torch.multinomial(weight, rows - used, replacement=True, generator=gen) if rows > used else who[:0]
    counts = torch.zeros(experts, device="cuda", dtype=torch.long)
    counts[who] = 1 + torch.bincount(more, minlength=used)
    return counts.cumsum(0).int(), int(counts.max())


def _parents(gen, sentences, beams, moved):
    """For `moved` of a sentence's beams another one, for the others themselves."""
    own_place = torch.arange(beams, device="cuda").expand(sentences, beams)
    other = (own_place + torch.randint(1, beams, (sentences, beams), device="cuda", generator=gen)) % beams
    order = torch.rand((sentences, beams), device="cuda", generator=gen).argsort(1)
    return torch.where(order < moved, other, own_place).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rand = functools.partial(torch.randn, device="cuda", generator=gen)
    op = case["op"]
    if op == "linear":
        w, w_scales = _weights(lambda *shape: rand(shape), case["n"], case["k"])
        return dict(op=op, x=_activations(gen, case["m"], case["k"], DTYPES[case["dtype"]]), w=w, w_scales=w_scales,
                    bias=rand(case["n"]) if case["bias"] else None)
    if op == "experts":
        whole = case["dtype"] == "int8"
        shape = case["experts"], case["n"], case["k"]
        w, w_scales = _weights(lambda *shape: rand(shape), *shape) if whole else (rand(shape).mul_(0.02).to(DTYPES[case["dtype"]]), None)
        ends, longest = _ends(gen, case["m"], case["experts"], case["used"])
        return dict(op=op, x=_activations(gen, case["m"], case["k"], torch.bfloat16 if whole else DTYPES[case["dtype"]]), w=w, w_scales=w_scales,
                    ends=ends, longest=longest, bias=rand((case["experts"], case["n"])) if case["bias"] else None)
    if op == "beams":
        sentences, beams, vocab = case["sentences"], case["beams"], case["vocab"]
        rows = sentences * beams
        logits = rand((rows, vocab)).mul_(2.5)
        if case["masked"]:
            logits.masked_fill_(torch.rand((rows, vocab), device="cuda", generator=gen) < case["masked"], -math.inf)
        third = vocab // 3      # a few tokens more probable than most
        likely = torch.randint(0, third, (rows, 3), device="cuda", generator=gen) + third * torch.arange(3, device="cuda")
        logits.scatter_(1, likely, 8 + 4 * torch.rand((rows, 3), device="cuda", generator=gen))
        ended = None
        if case["ended"]:
            ended = torch.rand((sentences, beams), device="cuda", generator=gen).argsort(1) < case["ended"]
        scores = -20 * torch.rand((sentences, beams), device="cuda", generator=gen)
        return dict(op=op, logits=logits.to(DTYPES[case["dtype"]]), scores=scores.sort(1, descending=True).values.contiguous(), select=case["select"],
                    ended=ended, end_token=2, scale=1.25)
    rows, dtype = case["sentences"] * case["beams"], DTYPES[case["dtype"]]
    cache = torch.empty((case["states"], rows, case["heads"], case["positions"], case["channels"]), device="cuda", dtype=dtype)
    cache.normal_(generator=gen)
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    lengths = lengths[torch.randperm(case["sentences"], device="cuda", generator=gen)]
    return dict(op=op, cache=cache, layers=list(cache.unbind(0)), lengths=lengths, parents=_parents(gen, case["sentences"], case["beams"], case["moved"]))


def _lengths(case):
    """From half of the positions to all but one, the same ones for every seed, in another order."""
    n, p = case["sentences"], case["positions"]
    return [max(1, (p + 1) // 2 + (p - 1 - (p + 1) // 2) * i // max(1, n - 1)) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "linear":
        m, n, k, es = case["m"], case["n"], case["k"], SIZES[case["dtype"]]
        return {"bytes": m * k * es + n * k + m * n * es + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    if op == "experts":
        m, n, k, es = case["m"], case["n"], case["k"], SIZES[case["dtype"]]
        per_channel = (4 if es == 1 else 0) + (4 if case["bias"] else 0)
        return {"bytes": 2 * m * (k + n) + case["used"] * n * (k * es + per_channel), "flops": 2 * m * n * k}
    if op == "beams":
        n = case["sentences"] * (case["beams"] - case["ended"]) * case["vocab"]
        return {"bytes": n * SIZES[case["dtype"]] + case["sentences"] * (5 * case["beams"] + 12 * case["select"]), "flops": 4 * n}
    moved = sum(_lengths(case)) * case["moved"] * case["states"] * case["heads"] * case["channels"] * SIZES[case["dtype"]]
    return {"bytes": 2 * moved + 8 * case["sentences"] * case["beams"], "flops": 0}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_rows(x):
    """Scales and their reciprocals are fp32 numbers; between them nothing is rounded."""
    largest = torch.linalg.vector_norm(x.double(), ord=math.inf, dim=1)
    scales = torch.maximum(largest / 127.0, largest.new_tensor(SMALLEST_SCALE)).float().double()
    return torch.round(x.double() * (1.0 / scales).float().double()[:, None]), scales


def exact(case, seed):
    if case["op"] == "reorder":
        return None      # copies
    s = prepare(case, seed)
    if s["op"] == "linear":
        q, scales = _exact_rows(s["x"])
        y = torch.einsum("mk,nk->mn", q, s["w"].double()) * scales[:, None] * s["w_scales"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    if s["op"] == "experts":
        q, scales = _exact_rows(s["x"]) if s["w_scales"] is not None else (s["x"].double(), None)
        out, first = [], 0
        for e, end in enumerate(s["ends"].tolist()):
            y = torch.einsum("mk,nk->mn", q[first:end], s["w"][e].double())
            if scales is not None:
                y = y * scales[first:end, None] * s["w_scales"][e].double()
            out.append(y if s["bias"] is None else y + s["bias"][e].double())
            first = end
        return torch.cat(out)
    got, parents, tokens = [], [], []
    sentences, beams = s["scores"].shape
    for i in range(sentences):
        found = []
        for j in range(beams):
            before = float(s["scores"][i, j])
            if s["ended"] is not None and bool(s["ended"][i, j]):
                found.append((-before, j, 0, s["end_token"]))
                continue
            z = s["logits"][i * beams + j].double() * s["scale"]
            values, order = z.sort(descending=True, stable=True)
            lse = torch.logsumexp(z, 0)
            each = (before + values[:case["select"]] - lse).tolist()
            found += [(-v, j, k, t) for k, (v, t) in enumerate(zip(each, order[:case["select"]].tolist())) if v > -math.inf]
        found = sorted(found)[:case["select"]]
        found += [(math.inf, -1, 0, -1)] * (case["select"] - len(found))
        got.append([-f[0] for f in found])
        parents.append([f[1] for f in found])
        tokens.append([f[3] for f in found])
    return torch.tensor(got, dtype=torch.float64), torch.tensor(parents, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
