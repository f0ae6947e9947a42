"""An int8 head, a block by experts and beam search run together."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _mods():
    import torch
    from excalibur_b200 import capi
    return torch, capi


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("rows,C,V", [(1, 512, 4001), (70, 1000, 1000), (300, 256, 9000)])
def test_token_head_in_integers(ctx, rows, C, V):
    torch, capi = _mods()
    from excalibur_b200.token_head import TokenHead
    g = _gen(rows)
    vocab = (torch.randn((V, C), device="cuda", generator=g) * 0.1).half()
    w = 1 + 0.1 * torch.randn(C, device="cuda", generator=g)
    head = TokenHead(ctx, vocab, w, residual_scale=0.5, weights="int8")
    h, x = torch.randn((rows, C), device="cuda", generator=g).half(), torch.randn((rows, C), device="cuda", generator=g).half()
    tokens = torch.randint(0, V, (rows, 2), device="cuda", generator=g).int()
    r, logits = head.logits(h, x)
    r2, n = capi.residual_norm(ctx, h, x, residual_scale=0.5, weight=w)
    q, s = capi.quantize_rows(ctx, n)
    again = capi.int8_matmul(ctx, q, s, head.weights, head.scales, out_dtype=capi.EXB_F32)
    given = head.scores(h, x, tokens, top=5)
    want = capi.token_logprobs(ctx, logits, tokens, top=5)
    ctx.sync_check()
    assert torch.equal(r, r2) and torch.equal(logits, again) and all(torch.equal(a, b) for a, b in zip(given, want))
    # against the same without 8 bits: an operand is off by up to half a step, 1 in 254 of its row's largest (about 3.5 times the row's spread), evenly spread:
    # 3.5 / 127 / sqrt(12) = 0.8 % of the spread each, which random signs leave as 0.8 % of a result's; two operands: 1.1 %
    ref = x.double() + 0.5 * h.double()
    ref = ref * (ref.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w.double()
    full = ref @ vocab.double().t()
    assert ((logits.double() - full).norm() / full.norm()) < 0.02
    with pytest.raises(ValueError):
        TokenHead(ctx, vocab, w, weights="int4")


@pytest.mark.parametrize("weights,dtype,tolerance", [("int8", "float16", 0.04), ("int8", "bfloat16", 0.05), ("own", "float16", 0.004), ("own", "bfloat16", 0.03)])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 2), (150, 2), (700, 4)])
def test_experts(ctx, weights, dtype, tolerance, rows, k):
    """Against the block in 64 bits: in integers each of four operands is off by about 0.8 % of its spread, in the types' own by half a step of a few roundings."""
    torch, capi = _mods()
    from excalibur_b200.experts import Experts
    t, E, C, H = getattr(torch, dtype), 6, 264, 200
    g = _gen(rows + k)
    up = (torch.randn((E, H, C), device="cuda", generator=g) * C ** -0.5).to(t)
    down = (torch.randn((E, C, H), device="cuda", generator=g) * H ** -0.5).to(t)
    x = torch.randn((rows, C), device="cuda", generator=g).to(t)
    scores = torch.randn((rows, E), device="cuda", generator=g)
    scores[:, 3] = -100.0                      # an expert without a row
    gates, chosen = torch.softmax(scores, 1).topk(k, 1)
    y = Experts(ctx, up, down, weights)(x, chosen, gates)
    ctx.sync_check()
    ref = torch.zeros((rows, C), device="cuda", dtype=torch.float64)
    for j in range(k):
        W1, W2 = up[chosen[:, j]].double(), down[chosen[:, j]].double()
        h = torch.nn.functional.silu(torch.einsum("rhc,rc->rh", W1, x.double()))
        ref += gates[:, j].double()[:, None] * torch.einsum("rch,rh->rc", W2, h)
    assert y.dtype == t and ((y.double() - ref).norm() / ref.norm()) < tolerance
    with pytest.raises(ValueError):
        Experts(ctx, up, down, "e4m3")


def test_beam_search_finds_what_an_exhaustive_one_does(ctx):
    """A decoder whose logits hang on the last token alone, with as many beams as there are tokens: every sequence of two is among the beams, and those of three are
    right by the states that follow them."""
    torch, capi = _mods()
    from excalibur_b200.beam_search import BeamSearch
    V, B, beams, steps = 7, 3, 32, 3
    table = torch.randn((B, V + 1, V), device="cuda", generator=_gen(1), dtype=torch.float64)
    lp = torch.log_softmax(table.float().double(), 2)
    search = BeamSearch(ctx, B, beams, end_token=0, most_tokens=steps)
    last = torch.full((B * beams, 1), V, device="cuda")                  # a state: each beam's last token
    which = torch.arange(B, device="cuda").repeat_interleave(beams)
    for _ in range(steps):
        tokens = search.step(table.float()[which, last[:, 0]].contiguous(), [last])
        assert (tokens.view(B, beams) == -1).equal(search.scores == -math.inf)
        last[:, 0] = tokens.clamp_min(0).long()
    ctx.sync_check()
    for b in range(B):
        found = {}
        for i in range(V):
            for j in range(V):
                for k in range(V):
                    if i == 0 and (j or k) or j == 0 and k:
                        continue
                    s = lp[b, V, i] + (0 if i == 0 else lp[b, i, j]) + (0 if j == 0 else lp[b, j, k])
                    found[(i, j, k)] = float(s)
        got = {tuple(t): s for t, s in zip(search.tokens.view(B, beams, -1)[b].tolist(), search.scores[b].tolist())}
        assert len(got) == beams
        for t, s in got.items():
            assert abs(found[t] - s) < 1e-5, (t, s)
        # (two tokens make 43 sequences of which 32 were kept, so that the 20 best of three may be checked for sure only where their beginnings were)
        best = sorted(found.items(), key=lambda z: -z[1])[:5]
        assert [t for t, _ in best] == [t for t, _ in sorted(got.items(), key=lambda z: -z[1])[:5]]
    assert len(search.best()[0]) == B
    with pytest.raises(ValueError):
        search.step(table.float()[which, last[:, 0]].contiguous())


def test_states_follow_their_beams_through_a_search(ctx):
    """A cache that holds what each beam has chosen, position by position, is the history of the tokens at every step."""
    torch, capi = _mods()
    from excalibur_b200.beam_search import BeamSearch
    B, beams, V, T = 4, 5, 300, 12
    search = BeamSearch(ctx, B, beams, end_token=5, most_tokens=T)
    caches = [torch.full((B * beams, 2, T, 8), -1.0, device="cuda").half() for _ in range(3)]
    g = _gen(2)
    for step in range(T):
        logits = torch.randn((B * beams, V), device="cuda", generator=g) * 3
        lengths = torch.full((B,), step, device="cuda", dtype=torch.int32)
        tokens = search.step(logits, caches, lengths)
        for i, c in enumerate(caches):
            c[:, :, step] = (tokens.half() + i)[:, None, None]
        for i, c in enumerate(caches):
            want = (search.tokens[:, :step + 1].half() + i)[:, None, :, None].expand(-1, 2, -1, 8)
            assert torch.equal(c[:, :, :step + 1], want)
        if step:
            assert (search.scores[:, 1:] <= search.scores[:, :-1]).all()
    ctx.sync_check()
    for row, ended in zip(search.tokens.tolist(), search.ended.view(-1).tolist()):
        assert (5 in row) == ended and (not ended or set(row[row.index(5):]) == {5})


@pytest.mark.parametrize("weights", ["int8", "e4m3"])
def test_the_command_runs(ctx, capsys, monkeypatch, weights):
    from excalibur_b200 import beam_search
    monkeypatch.setattr("sys.argv", ["beam_search", "--sentences", "3", "--beams", "3", "--channels", "128", "--vocab", "1000", "--steps", "5", "--experts", "4",
                                     "--weights", weights])
    beam_search.main()
    lines = capsys.readouterr().out.strip().split("\n")
    assert len(lines) == 3 and all(line.startswith("sentence %d: -" % i) for i, line in enumerate(lines))


def test_the_head_command_runs_in_integers(ctx, capsys, monkeypatch):
    from excalibur_b200 import token_head
    monkeypatch.setattr("sys.argv", ["token_head", "--rows", "3", "--channels", "256", "--vocab", "1000", "--top", "2", "--weights", "int8"])
    token_head.main()
    assert len(capsys.readouterr().out.strip().split("\n")) == 3
