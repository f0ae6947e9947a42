"""Beam search's selection and the reordering of states, against plain implementations in 64 bits, at the sizes, masks, strides and orders where they can go
wrong."""
import math

import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float16", "bfloat16", "float32")


def _mods():
    import torch
    from excalibur_b200 import capi
    return torch, capi


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- selection -----------------------------------------------------------------------------------------------------------

def _ref_scores(logits, scores, ended, end_token, scale):
    """Every candidate's score in 64 bits: (sentences, beams, V); minus infinity is none."""
    import torch
    sentences, beams = scores.shape
    x = logits.double().view(sentences, beams, -1)
    z = x * torch.tensor(scale, dtype=torch.float32).double().item()
    z = z - z.amax(2, keepdim=True)      # (64 bits do not hold a logarithm beside a type's lowest value)
    s = scores.double()[..., None] + (z - z.exp().sum(2, keepdim=True).log())
    bad = (torch.isnan(x) | (x == math.inf)).any(2, keepdim=True)
    s = torch.where(bad, math.nan, torch.where(x == -math.inf, -math.inf, s))
    if ended is not None:
        stay = torch.full_like(s, -math.inf)
        stay[..., end_token] = scores.double()
        s = torch.where(ended.bool()[..., None], stay, s)
    return torch.where(scores[..., None] == -math.inf, -math.inf, s)


def _tolerance(logits, scale):
    """Of a score: a thread or lane adds at most V / 32 exponentials one after the other and what it joins, each addition and each exponential off by 2^-23 of the sum
    and of itself at most; the scale times log2(e) is rounded, by 2^-23 of a distance from the largest, which weighs as e^-distance (times itself, below 1)."""
    return (logits.shape[1] / 32 + 200) * 2.0 ** -23


def _check(got, ref, logits, scale, select):
    """Every place's score is that candidate's, places fall, and no better candidate is left out - up to the tolerance, and rounding to fp32."""
    import torch
    out, parents, tokens = got
    sentences, beams, V = ref.shape
    tol = _tolerance(logits, scale)
    assert out.shape == parents.shape == tokens.shape == (sentences, select)
    best = ref.reshape(sentences, -1).sort(1, descending=True).values[:, :select]
    if best.shape[1] < select:
        best = torch.nn.functional.pad(best, (0, select - best.shape[1]), value=-math.inf)
    none = best == -math.inf
    assert torch.equal(out == -math.inf, none)
    assert torch.equal(parents == -1, none) and torch.equal(tokens == -1, none)
    flat = (parents.long() * V + tokens.long()).clamp_min(0)
    assert (parents < beams).all() and (tokens < V).all()
    for i in range(sentences):      # no candidate twice
        mine = flat[i][~none[i]]
        assert mine.unique().numel() == mine.numel()
    own = torch.where(none, -math.inf, ref.reshape(sentences, -1).gather(1, flat))
    fine = ~none
    near = tol + own[fine].abs() * 2.0 ** -23
    assert ((out.double()[fine] - own[fine]).abs() <= near).all(), float((out.double()[fine] - own[fine]).abs().max())
    assert (own[fine] - best[fine] >= -2 * tol).all() and (own[fine] - best[fine] <= 2 * tol).all()
    assert (out[:, 1:] <= out[:, :-1]).all()


def _logits(rows, V, dtype, seed, spread=2.5):
    import torch
    return (torch.randn((rows, V), device="cuda", generator=_gen(seed)) * spread).to(getattr(torch, dtype))


@pytest.mark.parametrize("sentences,beams,V,select", [
    (1, 1, 1, 1), (1, 1, 5, 8), (1, 4, 3, 12), (2, 3, 7, 32), (5, 2, 100, 4), (3, 5, 1000, 10), (300, 4, 1025, 8), (2, 32, 2000, 32), (64, 8, 333, 16), (7, 4, 4096, 4),
    (1, 4, 8191, 8), (33, 3, 10001, 6), (2, 16, 16384, 32), (1, 4, 50001, 8), (20, 5, 50001, 10), (1, 1, 131072, 1), (1, 8, 131072, 16), (100, 4, 20000, 8), (1, 4, 262144, 20)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_beam_select(ctx, sentences, beams, V, select, dtype):
    torch, capi = _mods()
    g = _gen(V + beams)
    logits = _logits(sentences * beams, V, dtype, V + select)
    scores = -20 * torch.rand((sentences, beams), device="cuda", generator=g)
    ended = torch.rand((sentences, beams), device="cuda", generator=g) < 0.2
    for scale, e in ((1.0, None), (1.25, ended)):
        end = min(2, V - 1)
        got = capi.beam_select(ctx, logits, scores, select, scale=scale, ended=e, end_token=end)
        again = capi.beam_select(ctx, logits, scores, select, scale=scale, ended=e, end_token=end)
        ctx.sync_check()
        _check(got, _ref_scores(logits, scores, e, end, scale), logits, scale, select)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 1000, 9000, 50003])
def test_beam_select_with_masks(ctx, dtype, V):
    """Half and nearly all of the tokens masked, whole rows, whole sentences; by minus infinity, and by the type's lowest value, which is a token like others."""
    torch, capi = _mods()
    B, beams, select = 6, 4, 8
    logits = _logits(B * beams, V, dtype, V)
    keep = torch.rand((B * beams, V), device="cuda", generator=_gen(1))
    for low in (-math.inf, torch.finfo(logits.dtype).min):
        x = logits.clone()
        x[keep < 0.5] = low
        x[:8][keep[:8] < 1 - 3 / V] = low        # a few tokens a row
        x[8:10] = low                             # rows without any
        x[12:16] = low                            # a sentence without any
        x[16, :] = low
        x[16, V - 1] = 1
        scores = -5 * torch.rand((B, beams), device="cuda", generator=_gen(2))
        got = capi.beam_select(ctx, x, scores, select)
        ctx.sync_check()
        _check(got, _ref_scores(x, scores, None, 0, 1.0), x, 1.0, select)
        if low == -math.inf:
            assert (got[1][3] == -1).all()


def test_beam_select_of_beams_that_are_none_or_have_ended(ctx):
    """Their rows are not read: they hold NaN.  The first step of a search has one beam."""
    torch, capi = _mods()
    for V, dtype in ((500, "float16"), (33333, "bfloat16"), (131072, "float32")):
        logits = _logits(8, V, dtype, V).view(2, 4, V)
        scores = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf], [-1.0, -2.0, -math.inf, -1.5]], device="cuda")
        ended = torch.tensor([[False, False, True, False], [True, False, True, True]], device="cuda")
        logits[0, 1:] = math.nan
        logits[1, 0] = logits[1, 2] = logits[1, 3] = math.nan
        got = capi.beam_select(ctx, logits.view(8, V), scores, 6, ended=ended, end_token=7)
        ctx.sync_check()
        _check(got, _ref_scores(torch.nan_to_num(logits.view(8, V)), scores, ended, 7, 1.0), logits, 1.0, 6)
        assert (got[1][0] == 0).all()
        assert [int(p) for p in got[1][1][:2]] == [0, 3] and [int(t) for t in got[2][1][:2]] == [7, 7] and got[0][1][:2].tolist() == [-1.0, -1.5]
        all_ended = capi.beam_select(ctx, logits.view(8, V), scores, 3, ended=torch.ones_like(ended).to(torch.uint8), end_token=V - 1)
        nothing = capi.beam_select(ctx, logits.view(8, V), torch.full_like(scores, -math.inf), 3)
        ctx.sync_check()
        assert all_ended[1].tolist() == [[0, -1, -1], [0, 3, 1]] and all_ended[2].tolist() == [[V - 1, -1, -1], [V - 1] * 3]
        assert (nothing[0] == -math.inf).all() and (nothing[1] == -1).all() and (nothing[2] == -1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [64, 3000, 60000])
def test_beam_select_of_equal_scores(ctx, dtype, V):
    """Equal rows have equal sums: the lower beam first, in a beam the larger logit, of equal ones the lower token."""
    torch, capi = _mods()
    row = torch.randint(-3, 3, (V,), device="cuda", generator=_gen(V)).to(getattr(torch, dtype))
    row[V // 2], row[V // 3], row[V - 1] = 4, 4, 4
    logits = row.expand(8, V).contiguous()
    scores = torch.zeros((2, 4), device="cuda")
    scores[1, 0] = -0.5
    got = capi.beam_select(ctx, logits, scores, 16)
    ctx.sync_check()
    order = row.double().sort(descending=True, stable=True)
    four, three = [V // 3, V // 2, V - 1], [int(t) for t in order.indices[3:16]]
    assert got[1][0].tolist()[:12] == [0] * 3 + [1] * 3 + [2] * 3 + [3] * 3 and got[2][0].tolist()[:12] == four * 4
    n = int((row == 2).sum())
    assert got[1][0].tolist()[12:] == [0] * min(4, n) + [1] * (4 - min(4, n)) and got[2][0].tolist()[12:12 + min(4, n)] == three[:min(4, n)]
    assert got[1][1].tolist()[:12] == [1] * 3 + [2] * 3 + [3] * 3 + [0] * 3 and got[2][1].tolist()[:12] == four * 4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 2500, 40000])
def test_beam_select_with_numbers_that_are_none(ctx, dtype, V):
    """A NaN or plus infinity in a row makes its scores NaN, which come first, the NaN token before the others; a score of plus infinity comes before finite ones."""
    torch, capi = _mods()
    for value in (math.nan, math.inf):
        logits = _logits(8, V, dtype, V)
        logits[5, V // 2] = value
        scores = torch.zeros((2, 4), device="cuda")
        scores[0, 3] = math.inf
        got = capi.beam_select(ctx, logits, scores, 4)
        ctx.sync_check()
        assert (got[1][0] == 3).all() and (got[0][0] == math.inf).all()
        assert (got[1][1] == 1).all() and torch.isnan(got[0][1]).all() and int(got[2][1, 0]) == V // 2
        assert got[2][0].tolist() == logits[3].double().sort(descending=True, stable=True).indices[:4].tolist()
    scores[1, 0] = math.nan
    got = capi.beam_select(ctx, torch.zeros_like(logits), scores, 4)
    ctx.sync_check()
    assert got[1][1].tolist() == [0] * 4 and got[2][1].tolist() == [0, 1, 2, 3] and torch.isnan(got[0][1]).all()


def test_beam_select_at_the_ends_of_scales_and_strides(ctx):
    torch, capi = _mods()
    for dtype in DTYPES:
        for V in (999, 20001):
            wide = torch.full((12, V + 13), math.nan, device="cuda", dtype=getattr(torch, dtype))
            x = wide[:, 5:5 + V]
            x.copy_(_logits(12, V, dtype, V))
            scores = -torch.rand((4, 3), device="cuda", generator=_gen(3)) * 1e4
            for scale in (1e-6, 0.1, 30.0, 1e5):
                got = capi.beam_select(ctx, x, scores, 7, scale=scale)
                ctx.sync_check()
                ref = _ref_scores(x, scores, None, 0, scale)
                out, parents, tokens = got
                # (a scaled distance from the largest logit is rounded as a whole: 2^-23 of what a selected score lies below its row's best)
                best = ref.amax(2)
                own = ref.view(4, -1).gather(1, parents.long() * V + tokens.long())
                near = _tolerance(x, scale) + own.abs() * 2.0 ** -22
                assert ((out.double() - own).abs() <= near).all()
                top = ref.view(4, -1).sort(1, descending=True).values[:, :7]
                assert ((own - top).abs() <= 2 * near).all() and torch.isfinite(best).all()


# ---- states ----------------------------------------------------------------------------------------------------------------

def _ref_reorder(state, parents, lengths):
    import torch
    sentences, beams = parents.shape
    new = state.clone()
    for i in range(sentences):
        for j in range(beams):
            p = int(parents[i, j])
            if 0 <= p < beams:
                if lengths is None:
                    new[i * beams + j] = state[i * beams + p]
                else:
                    n = max(0, int(lengths[i]))
                    new[i * beams + j, ..., :n, :] = state[i * beams + p, ..., :n, :]
    return new


def _bytes(t):
    import torch
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("sentences,beams", [(1, 1), (1, 2), (1, 4), (3, 4), (2, 5), (5, 8), (2, 13), (1, 16), (2, 17), (1, 32), (300, 3)])
@pytest.mark.parametrize("shape,dtype", [((2, 40, 64), "float16"), ((3, 17, 33), "float16"), ((1, 129, 80), "bfloat16"), ((4, 9, 5), "int8"), ((2, 33, 6), "float32"),
                                         ((2, 2, 31, 64), "float16")])
def test_reorder_beams(ctx, sentences, beams, shape, dtype):
    torch, capi = _mods()
    g = _gen(sentences * 100 + beams)
    rows = sentences * beams
    size = max(1, torch.empty(0, dtype=getattr(torch, dtype)).element_size())
    states = [torch.randint(0, 256, (rows, *shape[:-1], shape[-1] * size), device="cuda", generator=g, dtype=torch.int32).to(torch.uint8).view(getattr(torch, dtype))
              for _ in range(3)]
    parents = torch.randint(0, beams, (sentences, beams), device="cuda", generator=g, dtype=torch.int32)
    parents[0, beams - 1] = -1
    if sentences > 1:
        parents[1] = torch.arange(beams)         # nothing to do
        parents[sentences - 1, 0] = beams        # no beam's
    lengths = torch.randint(0, shape[-2] + 2, (sentences,), device="cuda", generator=g, dtype=torch.int32)
    lengths[0] = shape[-2] // 2
    for by in (lengths, None):
        want = [_ref_reorder(s, parents, by) for s in states]
        mine = [s.clone() for s in states]
        capi.reorder_beams(ctx, mine, parents, by)
        ctx.sync_check()
        for a, b in zip(mine, want):
            assert torch.equal(_bytes(a), _bytes(b))


def test_reorder_beams_of_lengths_at_the_ends(ctx):
    torch, capi = _mods()
    state = torch.randn((12, 3, 20, 16), device="cuda", generator=_gen(1)).half()
    parents = torch.tensor([[1, 2, 0]] * 4, dtype=torch.int32, device="cuda")
    for lengths in ([0, 1, 20, 21], [-5, 2 ** 31 - 1, -2 ** 31, 19], [0, 0, 0, 0]):
        at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want, mine = _ref_reorder(state, parents, at), state.clone()
        capi.reorder_beams(ctx, mine, parents, at)
        ctx.sync_check()
        assert torch.equal(mine, want)


def test_reorder_beams_takes_strides_and_leaves_the_rest(ctx):
    """Views of one buffer: heads inside positions, layers inside rows, keys beside values, part of the positions or channels, rows that start anywhere."""
    torch, capi = _mods()
    B, beams, H, T, D = 3, 4, 2, 24, 16
    rows = B * beams
    parents = torch.tensor([[3, 0, 0, 1], [0, 1, 2, 3], [2, 2, 2, 0]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([7, 24, 13], dtype=torch.int32, device="cuda")
    g = _gen(7)

    def fresh(*shape):
        return torch.randn(shape, device="cuda", generator=g).half()
    for make in (lambda w: [w.transpose(1, 2)], lambda w: [w[:, :, 3:20]], lambda w: [w[..., 8:]], lambda w: [w[..., 3:10]], lambda w: [w[:, 1]],
                 lambda w: [w[..., :8], w[..., 8:]], lambda w: [w[:, :1], w[:, 1:]], lambda w: [w[:, :, ::2], w[:, :, 1::2]]):
        for by in (lengths, None):
            whole = fresh(rows, H, T, D)
            mine = whole.clone()
            views = make(mine)
            for v, w in zip(views, make(whole)):
                w.copy_(_ref_reorder(w.clone(), parents, by))
            capi.reorder_beams(ctx, views, parents, by)
            ctx.sync_check()
            assert torch.equal(mine, whole)
    layers = fresh(rows, 5, H, T, D)      # layers inside rows
    want = _ref_reorder(layers, parents, lengths)
    capi.reorder_beams(ctx, list(layers.unbind(1)), parents, lengths)
    ctx.sync_check()
    assert torch.equal(layers, want)


def test_reorder_beams_of_states_unlike_each_other_and_of_many(ctx):
    torch, capi = _mods()
    parents = torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    g = _gen(3)
    states = [torch.randn((4, 3, 10, 8), device="cuda", generator=g).half(), torch.randn((4, 5), device="cuda", generator=g),
              torch.randint(0, 99, (4,), device="cuda", generator=g), torch.empty((4, 0), device="cuda"), torch.randn((4, 3, 10, 8), device="cuda", generator=g)]
    want = [_ref_reorder(s, parents, None) for s in states]
    capi.reorder_beams(ctx, states, parents)
    ctx.sync_check()
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    many = [torch.randn((4, 2, 6, 4), device="cuda", generator=g) for _ in range(300)]
    want = [_ref_reorder(s, parents, None) for s in many]
    capi.reorder_beams(ctx, many, parents)
    capi.reorder_beams(ctx, [], parents)
    ctx.sync_check()
    assert all(torch.equal(a, b) for a, b in zip(many, want))


def test_reorder_beams_refuses_before_anything_moves(ctx):
    torch, capi = _mods()
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    state = torch.randn((2, 3, 4), device="cuda")
    before = state.clone()
    for bad in (state, state[:, :2], torch.randn((1, 5), device="cuda").expand(2, 5), torch.randn((3, 5), device="cuda"), torch.randn((2, 5))):
        with pytest.raises(capi.ExbError):
            capi.reorder_beams(ctx, [state, bad], parents)
    ctx.sync_check()
    assert torch.equal(state, before)


# ---- together --------------------------------------------------------------------------------------------------------------

def test_streams_and_graphs(ctx):
    """A captured step (selection, then the states follow) that is replayed, on another stream, two graphs in turn."""
    torch, capi = _mods()
    B, beams, V = 3, 4, 5000
    xs = [_logits(B * beams, V, "float16", i) for i in range(3)]
    caches = [torch.randn((B * beams, 2, 16, 32), device="cuda", generator=_gen(i)).half() for i in range(3)]
    scores = -torch.rand((B, beams), device="cuda", generator=_gen(9))
    lengths = torch.tensor([3, 16, 9], dtype=torch.int32, device="cuda")

    def step(x, cache):
        got = capi.beam_select(ctx, x, scores)
        capi.reorder_beams(ctx, cache, got[1], lengths)
        return got
    want = []
    for x, c in zip(xs, caches):
        mine = c.clone()
        want.append((*step(x, mine), mine))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    mine = caches[1].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = step(xs[1], mine)
        ctx.sync_check()
    assert all(torch.equal(a, b) for a, b in zip((*got, mine), want[1]))
    graphs = []
    for _ in range(2):
        x, c = xs[0].clone(), caches[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, c)
        graphs.append((g, x, c, out))
    for turn in range(4):
        for i, (g, x, c, _) in enumerate(graphs):
            x.copy_(xs[(turn + i) % 3])
            c.copy_(caches[(turn + i) % 3])
            g.replay()
        torch.cuda.synchronize()
        for i, (_, _, c, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip((*out, c), want[(turn + i) % 3]))
    ctx.sync_check()


def test_another_device_than_the_contexts_is_refused(ctx):
    torch, capi = _mods()
    logits, scores = torch.randn((4, 100), device="cuda"), torch.zeros((2, 2), device="cuda")
    parents = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    for call in (lambda: capi.beam_select(ctx, logits.cpu(), scores), lambda: capi.beam_select(ctx, logits, scores.cpu()),
                 lambda: capi.beam_select(ctx, logits, scores, ended=torch.zeros((2, 2), dtype=torch.bool)), lambda: capi.reorder_beams(ctx, logits.cpu(), parents),
                 lambda: capi.reorder_beams(ctx, logits, parents.cpu()), lambda: capi.reorder_beams(ctx, logits[:, :, None], parents, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(capi.ExbError):
            call()
    ctx.sync_check()
