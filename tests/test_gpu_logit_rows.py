"""The largest tokens of rows of logits with masks, for log probabilities and beam selection alike, in the shortest rows that a CTA has (just above 2048 bytes): most
threads have one vector or none there, so that a mask of a few dozen tokens leaves whole groups of threads without a finite logit."""
import math

import pytest

pytestmark = pytest.mark.gpu

SHORT = [("float32", V) for V in (513, 515, 518)] + [(t, V) for t in ("float16", "bfloat16") for V in (1025, 1028, 1031, 1038)]


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _masked(dtype, V, seed):
    """64 rows, at every alignment: eight each with a block of 32 and of 100 masked tokens, with 10 tokens left (anywhere, and at the front), with the last 40 left, with a half
    masked, without a mask and with nothing left."""
    import torch
    g = _gen(seed)
    wide = torch.full((64, -(-V // 8) * 8 + 1), math.nan, device="cuda", dtype=getattr(torch, dtype))      # (rows 1 element further from 16 bytes each)
    x = torch.randn((64, V), device="cuda", generator=g) * 3
    for i in range(8):
        at = int(torch.randint(0, V - 100, (1,), device="cuda", generator=g))
        x[i, at:at + 32] = -math.inf
        x[8 + i, at:at + 100] = -math.inf
        few = torch.randperm(V, device="cuda", generator=g)[:V - 10]
        x[16 + i, few] = -math.inf
        x[24 + i, 10:] = -math.inf
        x[32 + i, :-40] = -math.inf
        x[40 + i, torch.rand(V, device="cuda", generator=g) < 0.5] = -math.inf
    x[56:] = -math.inf
    rows = wide[:, :V]
    rows.copy_(x)
    return rows


def _near(V, ref):
    """A thread or lane adds at most max(V / 256, 256) exponentials one after the other and 40 additions join them, each off by 2^-24; an exponential is off by 2^-22;
    distances from the largest logit weigh as p times themselves, ln V at most on the average, of which 2^-24 is lost a few times, as of the sum's logarithm: 2^-18 in
    all.  The result and the distance in it are rounded to fp32."""
    return (max(V / 256, 256) + 40) * 2.0 ** -24 + 2.0 ** -18 + ref.abs() * 2.0 ** -21


@pytest.mark.parametrize("top", [1, 16, 17, 20, 32])
@pytest.mark.parametrize("dtype,V", SHORT)
def test_most_probable_tokens_of_short_masked_rows(ctx, dtype, V, top):
    import torch
    from excalibur_b200 import capi
    x = _masked(dtype, V, V + top)
    got = torch.full((64, top), -7.0, device="cuda"), torch.full((64, top), -7, device="cuda", dtype=torch.int32)      # every place has to be written
    capi.check(capi.lib().exb_token_logprobs_fwd(ctx._h, capi._pack_logprobs(64, x.stride(0), V, capi.exb_dtype_of(x), 0, top, 1.0, 0), x.data_ptr(), None, None, None,
                                                 got[0].data_ptr(), got[1].data_ptr(), capi._stream()))
    ctx.sync_check()
    z, order = x.double().sort(dim=1, descending=True, stable=True)
    lp = torch.where(z[:, :top] == -math.inf, -math.inf, z[:, :top] - torch.logsumexp(z, 1, keepdim=True))
    assert torch.equal(got[1], order[:, :top].int())
    none = lp == -math.inf
    assert torch.equal(got[0] == -math.inf, none)
    assert ((got[0].double() - lp).abs()[~none] <= _near(V, lp[~none])).all()


@pytest.mark.parametrize("beams,select", [(4, 8), (4, 17), (1, 20), (4, 32), (16, 32), (32, 32)])
@pytest.mark.parametrize("dtype,V", SHORT)
def test_selection_from_short_masked_rows(ctx, dtype, V, beams, select):
    """In one kernel (up to 16 beams) and in two."""
    import torch
    from excalibur_b200 import capi
    x = _masked(dtype, V, V + select)
    sentences = 64 // beams
    order = torch.randperm(64, device="cuda", generator=_gen(beams))      # (rows of every kind in a sentence)
    wide = torch.empty((64, x.stride(0)), device="cuda", dtype=x.dtype)
    x = wide[:, :V].copy_(x[order])
    scores = -4 * torch.rand((sentences, beams), device="cuda", generator=_gen(5))
    out = torch.full((sentences, select), -7.0, device="cuda")
    parents, tokens = (torch.full((sentences, select), -7, device="cuda", dtype=torch.int32) for _ in range(2))
    room = 8 * 64 * (1 + select)
    workspace = torch.empty(room, device="cuda", dtype=torch.uint8)
    capi.check(capi.lib().exb_beam_select_fwd(ctx._h, capi._pack_beams(sentences, x.stride(0), room, beams, V, capi.exb_dtype_of(x), select, 0, 1.0), x.data_ptr(),
                                              scores.data_ptr(), None, out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), workspace.data_ptr(), capi._stream()))
    ctx.sync_check()
    z = x.double()
    each = torch.where(z == -math.inf, -math.inf, z - torch.logsumexp(z, 1, keepdim=True)).view(sentences, beams, V) + scores.double()[..., None]
    best, at = each.view(sentences, -1).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :select + 1], at[:, :select + 1]
    none = best[:, :select] == -math.inf
    assert torch.equal(out == -math.inf, none) and torch.equal(parents == -1, none) and torch.equal(tokens == -1, none)
    near = _near(V, best)
    assert ((out.double() - best[:, :select]).abs()[~none] <= near[:, :select][~none]).all()
    # the very candidates, wherever the one before and the one behind are further away than the sums may be off
    gap = torch.nan_to_num(best[:, :-1] - best[:, 1:], nan=0.0, posinf=math.inf) > 2 * near[:, :select]
    sure = gap & torch.cat([torch.ones_like(gap[:, :1]), gap[:, :-1]], 1) & ~none
    assert sure.float().mean() > 0.5 * (~none).float().mean()
    assert torch.equal((parents.long() * V + tokens.long())[sure], at[:, :select][sure])


def _sure(scores, parents, near, select):
    """The places that have to hold the reference's very candidate: the next score is further away than twice what sums may be off, or all that lie within that are one
    beam's, whose order is that of its logits."""
    sure, first = [False] * select, 0
    for i in range(1, len(scores) + 1):
        if i == len(scores) or scores[i - 1] - scores[i] > 2 * near:
            whole = i < len(scores) and len(set(parents[first:i])) == 1
            for k in range(first, min(i, select)):
                sure[k] = whole
            first = i
    return sure


@pytest.mark.parametrize("sentences,beams,V,select", [(1, 1, 50001, 32), (1, 4, 131072, 8), (1, 8, 262144, 16), (64, 5, 50001, 10), (2, 16, 131072, 32), (4, 32, 50000, 32),
                                                      (40, 8, 131072, 8), (300, 4, 2050, 20), (500, 4, 8000, 17), (700, 3, 1000, 32)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_selection_is_the_references_where_scores_are_apart(ctx, sentences, beams, V, select, dtype):
    """Scores within what sums and roundings may be off (4e-5 at 131072 tokens), and the reference's own candidates in its order."""
    import torch
    from excalibur_b200 import capi
    g = _gen(V + select)
    x = (torch.randn((sentences * beams, V), device="cuda", generator=g) * 2.5).to(getattr(torch, dtype))
    scores = -3 * torch.rand((sentences, beams), device="cuda", generator=g)
    got = capi.beam_select(ctx, x, scores, select)
    ctx.sync_check()
    more = select + 24
    rows = []
    for r in range(0, sentences * beams, 64):      # (the rows' best `more` are all that can be among a sentence's)
        z = x[r:r + 64].double()
        best, at = z.sort(dim=1, descending=True, stable=True)
        rows.append((best[:, :more] - torch.logsumexp(z, 1, keepdim=True), at[:, :more]))
    each, at = (torch.cat([row[k] for row in rows]).view(sentences, beams * more) for k in (0, 1))
    each = each + scores.double().repeat_interleave(more, 1)
    best, order = each.sort(dim=1, descending=True, stable=True)
    best, order = best[:, :more], order[:, :more]
    parents, tokens = order // more, at.gather(1, order)
    near = float(_near(V, torch.zeros(())))
    assert ((got[0].double() - best[:, :select]).abs() <= near + best[:, :select].abs() * 2.0 ** -21).all()
    sure = torch.tensor([_sure(s, p, near + 2.0 ** -21 * abs(s[-1]), select) for s, p in zip(best.tolist(), parents.tolist())], device="cuda")
    assert sure.float().mean() > 0.5
    assert torch.equal(got[1][sure].long(), parents[:, :select][sure]) and torch.equal(got[2][sure].long(), tokens[:, :select][sure])
