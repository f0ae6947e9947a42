"""Decoding in 8-bit integers, by experts and with beams: results where torch has no short way to device memory, and scales beyond what their product holds."""
import math

import pytest

pytestmark = pytest.mark.gpu


def test_results_are_the_same_by_torchs_public_allocation(ctx, monkeypatch):
    """With and without the private function that the binding takes room by where this torch has it: the same values, sizes and strides."""
    import torch
    from excalibur_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(8)
    x, w = torch.randn((40, 300), device="cuda", generator=g).half(), torch.randn((4, 72, 300), device="cuda", generator=g).half()
    ends = torch.tensor([9, 9, 31, 40], device="cuda", dtype=torch.int32)
    logits, scores = torch.randn((40, 700), device="cuda", generator=g), -torch.rand((2, 20), device="cuda", generator=g)      # (short rows: through a workspace)

    def everything():
        q, s = capi.quantize_rows(ctx, x)
        qw, sw = capi.quantize_rows(ctx, w.view(-1, 300))
        y = capi.int8_matmul(ctx, q, s, qw, sw, out_dtype=capi.EXB_F32)
        z = capi.grouped_matmul(ctx, q, qw.unflatten(0, (4, 72)), ends, s, sw.view(4, 72), out_dtype=capi.EXB_BF16)
        return [q, s, qw, sw, y, z, *capi.beam_select(ctx, logits, scores, 7), *capi.beam_select(ctx, logits[:4], scores[:1, :4].contiguous())]
    want = everything()
    monkeypatch.setattr(capi, "_EMPTY", None)
    got = everything()
    ctx.sync_check()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.dtype is b.dtype and a.stride() == b.stride()


@pytest.mark.parametrize("M", [1, 40, 700])
def test_scales_whose_product_is_no_ordinary_number(ctx, M):
    """Products of scales are rounded to fp32 on their own: infinite ones make infinities, of a sum of 0 NaN, and subnormal ones keep the bits that those have."""
    import torch
    from excalibur_b200 import capi
    g = torch.Generator(device="cuda").manual_seed(M)
    a, w = (torch.randint(-3, 4, (n, 64), device="cuda", generator=g, dtype=torch.int8) for n in (M, 96))
    a[0] = 0
    sums = (a.double() @ w.double().t())
    for row, channel in ((1e30, 1e30), (2.0 ** -100, 3.0 * 2.0 ** -44)):
        sa, sw = torch.full((M,), row, device="cuda"), torch.full((96,), channel, device="cuda")
        product = (sa[:, None] * sw).double()      # rounded once, as the definition says
        want = (sums * product).float()
        y = capi.int8_matmul(ctx, a, sa, w, sw, out_dtype=capi.EXB_F32)
        z = capi.grouped_matmul(ctx, a, w[None], torch.tensor([M], device="cuda", dtype=torch.int32), sa, sw[None], out_dtype=capi.EXB_F32)
        ctx.sync_check()
        for r in (y, z):
            assert torch.equal(torch.isnan(r), torch.isnan(want)) and torch.equal(torch.nan_to_num(r), torch.nan_to_num(want))
        assert math.isnan(float(y[0, 0])) == (row == 1e30)
