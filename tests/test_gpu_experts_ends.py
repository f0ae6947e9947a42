"""A feed-forward block by experts at the ends: no rows, no experts a row, one expert for all rows."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights,dtype", [("int8", "float16"), ("int8", "bfloat16"), ("int8", "float32"), ("own", "float16"), ("own", "bfloat16")])
@pytest.mark.parametrize("rows,k", [(0, 2), (3, 0), (0, 0), (1, 1)])
def test_experts_of_nothing(ctx, weights, dtype, rows, k):
    import torch
    from excalibur_b200.experts import Experts
    t, g = getattr(torch, dtype), torch.Generator(device="cuda").manual_seed(1)
    up, down = (torch.randn(shape, device="cuda", generator=g).mul_(0.1).to(t) for shape in ((3, 40, 24), (3, 24, 40)))
    x = torch.randn((rows, 24), device="cuda", generator=g).to(t)
    y = Experts(ctx, up, down, weights)(x, torch.zeros((rows, k), device="cuda", dtype=torch.long), torch.ones((rows, k), device="cuda"))
    ctx.sync_check()
    assert y.shape == (rows, 24) and y.dtype == t
    assert torch.isfinite(y).all() and (k or not y.any())
