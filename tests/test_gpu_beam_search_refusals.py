"""A step of beam search that is refused leaves the search, and every state, as they were."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_refused_step_is_no_step(ctx):
    import torch
    from excalibur_b200 import capi
    from excalibur_b200.beam_search import BeamSearch
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = [torch.randn((6, 50), device="cuda", generator=g) for _ in range(3)]
    searches = [BeamSearch(ctx, 2, 3, end_token=0, most_tokens=4) for _ in range(2)]
    caches = [torch.randn((6, 2, 4, 8), device="cuda", generator=g).half()]
    caches.append(caches[0].clone())
    for i, x in enumerate(logits):
        want = searches[0].step(x, [caches[0]])
        search, cache = searches[1], caches[1]
        bad = (lambda: search.step(x, [cache, cache]), lambda: search.step(x, [cache, torch.zeros((5, 2), device="cuda")]),
               lambda: search.step(x, [cache, cache.cpu()]), lambda: search.step(x[:5], [cache]), lambda: search.step(x, [cache], torch.zeros(3, device="cuda", dtype=torch.int32)))
        for call in bad:
            with pytest.raises(capi.ExbError):
                call()
        got = search.step(x, [cache])
        ctx.sync_check()
        assert torch.equal(got, want) and torch.equal(search.scores, searches[0].scores) and torch.equal(search.tokens, searches[0].tokens)
        assert torch.equal(search.ended, searches[0].ended) and search.length == i + 1 and torch.equal(cache, caches[0])
