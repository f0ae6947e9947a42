"""8-bit and grouped products, rows in 8 bits, beam selection and reordering at the ends: offsets beyond 32 bits, single elements, nothing at all, two streams at
once, other weights than the activations' in a row."""
import math

import pytest

from test_gpu_beams import _check, _ref_reorder, _ref_scores
from test_gpu_int8_experts import _check_float, _check_int8, _gen, _mods, _ref_rows

pytestmark = pytest.mark.gpu


def test_results_beyond_32_bits(ctx):
    """600 000 rows of 4096 results: 2.5e9 elements, rows at the beginning, in the middle and at the end."""
    torch, capi = _mods()
    M, N, K = 600000, 4096, 64
    a = torch.randint(-127, 128, (M, K), device="cuda", generator=_gen(1), dtype=torch.int32).to(torch.int8)
    w = torch.randint(-127, 128, (N, K), device="cuda", generator=_gen(2), dtype=torch.int32).to(torch.int8)
    sa, sw = torch.rand(M, device="cuda", generator=_gen(3)) * 1e-2, torch.rand(N, device="cuda", generator=_gen(4)) * 1e-2
    y = capi.int8_matmul(ctx, a, sa, w, sw)
    ctx.sync_check()
    for s in (slice(0, 300), slice(M // 2, M // 2 + 300), slice(524200, 524400), slice(M - 300, M)):
        _check_int8(y[s], a[s], sa[s], w, sw, None, "float16")
    x = y.view(-1, 65536)[:16000]            # rows in 8 bits out of more than 2^30 of them, in rows that are read twice
    q, scales = capi.quantize_rows(ctx, y[:, :3000])
    ctx.sync_check()
    for s in (slice(0, 50), slice(M - 50, M)):
        rq, rs = _ref_rows(y[s, :3000])
        assert torch.equal(q[s].cpu(), rq) and torch.equal(scales[s].cpu(), rs)
    q, scales = capi.quantize_rows(ctx, x)
    ctx.sync_check()
    rq, rs = _ref_rows(x[-5:])
    assert torch.equal(q[-5:].cpu(), rq) and torch.equal(scales[-5:].cpu(), rs)


def test_weights_beyond_32_bits(ctx):
    """130 experts of 4096 x 8192 in 8 bits: 4.4e9 bytes; the last ones' rows."""
    torch, capi = _mods()
    E, N, K = 130, 4096, 8192
    w = torch.empty((E, N, K), device="cuda", dtype=torch.int8)
    w.view(torch.int32).random_(generator=_gen(1))
    sw = torch.rand((E, N), device="cuda", generator=_gen(2)) * 1e-3
    for M in (3, 260, 1300):
        a = torch.randint(-127, 128, (M, K), device="cuda", generator=_gen(3), dtype=torch.int32).to(torch.int8)
        sa = torch.rand(M, device="cuda", generator=_gen(4)) * 1e-3
        ends = torch.zeros(E, device="cuda", dtype=torch.int32)
        ends[64:] = 1
        ends[128:] = M // 2
        ends[129] = M
        y = capi.grouped_matmul(ctx, a, w, ends, sa, sw, out_dtype=capi.EXB_F32)
        ctx.sync_check()
        for e, s in ((64, slice(0, 1)), (128, slice(1, M // 2)), (129, slice(M // 2, M))):
            if s.start < s.stop:
                _check_int8(y[s], a[s], sa[s], w[e], sw[e], None, "float32")


def test_logits_beyond_32_bits(ctx):
    torch, capi = _mods()
    for sentences, beams, V in ((2, 4, 1 << 28), (5000, 2, 250000)):
        logits = torch.empty((sentences * beams, V), device="cuda", dtype=torch.bfloat16)
        for row in logits.view(-1, min(V * beams, 1 << 28)) if V > 1 << 20 else [logits]:
            row.normal_(generator=_gen(1)) if row.dim() else None
        logits[-1, V - 1] = 30
        scores = -torch.rand((sentences, beams), device="cuda", generator=_gen(2))
        got = capi.beam_select(ctx, logits, scores, 4)
        ctx.sync_check()
        last = slice(sentences - 1, sentences)
        ref = _ref_scores(logits[-beams:], scores[last], None, 0, 1.0)
        _check([g[last] for g in got], ref, logits[-beams:], 1.0, 4)
        assert int(got[1][-1, 0]) == beams - 1 and int(got[2][-1, 0]) == V - 1
        del logits, ref


def test_states_beyond_32_bits(ctx):
    """Rows that start more than 2^32 bytes from the state's beginning, positions that do so within a row, vectors and single bytes."""
    torch, capi = _mods()
    parents = torch.tensor([[1, 0, 2, 2]], dtype=torch.int32, device="cuda")
    for size in (1 << 30, (1 << 30) + 3):
        state = torch.empty((4, size + 1300000000), device="cuda", dtype=torch.uint8)[:, :size]
        ends = torch.arange(4, device="cuda", dtype=torch.uint8)[:, None]
        for at in (slice(0, 64), slice(size // 2, size // 2 + 64), slice(size - 64, size)):
            state[:, at] = ends + 10
        capi.reorder_beams(ctx, state, parents)
        ctx.sync_check()
        for at in (slice(0, 64), slice(size // 2, size // 2 + 64), slice(size - 64, size)):
            assert (state[:, at].long() == torch.tensor([11, 10, 12, 12], device="cuda")[:, None]).all()
        del state
    state = torch.zeros((70000, 4, 4, 4096), device="cuda", dtype=torch.uint8).transpose(0, 2)      # (rows, 4, positions, 4096): positions far apart
    assert state.stride(2) * 69999 > 1 << 32
    state[:, :, :, 0] = torch.arange(4, device="cuda", dtype=torch.uint8)[:, None, None]
    capi.reorder_beams(ctx, state, parents, torch.tensor([69000], dtype=torch.int32, device="cuda"))
    ctx.sync_check()
    assert (state[:, :, :69000, 0].long() == torch.tensor([1, 0, 2, 2], device="cuda")[:, None, None]).all()
    assert (state[:, :, 69000:, 0].long() == torch.arange(4, device="cuda")[:, None, None]).all() and int(state[:, :, :, 1:9].max()) == 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_single_elements(ctx, dtype):
    torch, capi = _mods()
    t = getattr(torch, dtype)
    for M, N, K, E in ((1, 1, 1, 1), (1, 1, 3, 1), (1, 1, 9, 1), (1, 5, 8, 3), (5, 1, 8, 3)):
        a, w = torch.randn((M, K), device="cuda").to(t), torch.randn((E, N, K), device="cuda").to(t)
        ends = torch.full((E,), M, dtype=torch.int32, device="cuda")
        y = capi.grouped_matmul(ctx, a, w, ends)
        ctx.sync_check()
        _check_float(y, a, w[0], None, dtype)


def test_nothing_at_all(ctx):
    torch, capi = _mods()
    q, s = capi.quantize_rows(ctx, torch.empty((0, 100), device="cuda").half())
    w, sw = capi.quantize_rows(ctx, torch.randn((7, 100), device="cuda"))
    y = capi.int8_matmul(ctx, q, s, w, sw)
    z = capi.grouped_matmul(ctx, q, w[None], torch.zeros(1, dtype=torch.int32, device="cuda"), s, sw[None])
    b = capi.beam_select(ctx, torch.empty((0, 50), device="cuda"), torch.empty((0, 3), device="cuda"))
    capi.reorder_beams(ctx, torch.empty((0, 4), device="cuda"), torch.empty((0, 3), dtype=torch.int32, device="cuda"))
    capi.reorder_beams(ctx, torch.empty((3, 0, 4), device="cuda"), torch.zeros((1, 3), dtype=torch.int32, device="cuda"))
    ctx.sync_check()
    assert q.shape == (0, 100) and y.shape == z.shape == (0, 7) and all(v.shape == (0, 3) for v in b)


def test_two_streams_at_once(ctx):
    """Calls of every kernel under way on two streams, each against the same calls one after the other."""
    torch, capi = _mods()
    g = _gen(1)
    w, sw = capi.quantize_rows(ctx, torch.randn((3 * 700, 1024), device="cuda", generator=g))
    xs = [torch.randn((M, 1024), device="cuda", generator=g).half() for M in (3, 40, 90, 600)]
    logits, scores = torch.randn((24, 20000), device="cuda", generator=g), torch.zeros((6, 4), device="cuda")

    def work():
        out = []
        for x in xs:
            M = x.shape[0]
            q, s = capi.quantize_rows(ctx, x)
            out.append(capi.int8_matmul(ctx, q, s, w, sw))
            ends = torch.tensor([M // 3, M // 2, M], dtype=torch.int32).cuda()
            out.append(capi.grouped_matmul(ctx, q, w.view(3, 700, 1024), ends, s, sw.view(3, 700)))
            out.append(capi.grouped_matmul(ctx, x, w.view(3, 700, 1024).half(), ends, out_dtype=capi.EXB_F32))
        out += capi.beam_select(ctx, logits, scores, 8)
        cache = logits[:, :6400].clone().view(24, 4, 100, 16)
        capi.reorder_beams(ctx, cache, out[-2][:, :4].contiguous())
        return out + [cache]
    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for s, to in zip(streams, got):
            with torch.cuda.stream(s):
                to.append(work())
    torch.cuda.synchronize()
    ctx.sync_check()
    for runs in got:
        for out in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("M", [1, 30, 300])
def test_products_with_scales_at_the_ends(ctx, M):
    """Scales of rows and channels that span fp32, as long as their product is one of its normal numbers; zeros stay zeros.  (1 / scales: products of up to
    2^120, whose results of 2^128 and more no fp32 number is near: these are infinite.)"""
    torch, capi = _mods()
    a = torch.randint(-127, 128, (M, 200), device="cuda", generator=_gen(1), dtype=torch.int32).to(torch.int8)
    w = torch.randint(-127, 128, (64, 200), device="cuda", generator=_gen(2), dtype=torch.int32).to(torch.int8)
    pad_a, pad_w = torch.zeros((M, 208), device="cuda", dtype=torch.int8), torch.zeros((64, 208), device="cuda", dtype=torch.int8)
    pad_a[:, :200], pad_w[:, :200] = a, w
    w[5] = 0
    pad_w[5] = 0
    sa = torch.full((M,), 2.0 ** -100, device="cuda")
    sw = 2.0 ** (torch.arange(64, device="cuda") * 2.0 - 20)
    y = capi.int8_matmul(ctx, pad_a[:, :200], sa, pad_w[:, :200], sw, None, capi.EXB_F32)
    z = capi.int8_matmul(ctx, pad_a[:, :200], 1 / sa, pad_w[:, :200], 1 / sw, None, capi.EXB_F32)
    ctx.sync_check()
    _check_int8(y, a, sa, w, sw, None, "float32")
    ref = (a.double() @ w.double().t()) * (1 / sa).double()[:, None] * (1 / sw).double()
    beyond = ref.abs() >= 2.0 ** 128
    assert int(beyond.sum()) > 0 and (z[beyond].double() == torch.sign(ref[beyond]) * math.inf).all()
    keep = ~beyond.any(0)
    _check_int8(z[:, keep], a, 1 / sa, w[keep], (1 / sw)[keep], None, "float32")
    assert (y[:, 5] == 0).all() and (z[:, 5] == 0).all()


def test_the_workspace_is_for_the_calls_that_need_one(ctx):
    """More than 16 beams, short rows and many rows go through a workspace: refused without one, and the same answers with one."""
    torch, capi = _mods()
    import ctypes as C
    L = capi.lib()
    for sentences, beams, V in ((2, 17, 5000), (3, 4, 500), (600, 2, 9000), (2, 4, 5000)):
        logits, scores = torch.randn((sentences * beams, V), device="cuda", generator=_gen(V)), torch.zeros((sentences, beams), device="cuda")
        out = torch.full((3, sentences, 4), 7, device="cuda", dtype=torch.int32)

        def call(workspace, room):
            d = capi.BeamDesc(sentences=sentences, stride=V, workspace_bytes=room, beams=beams, V=V, dtype=capi.EXB_F32, select=4, end_token=0, scale=1.0)
            return L.exb_beam_select_fwd(ctx.handle, C.byref(d), logits.data_ptr(), scores.data_ptr(), None, *(o.data_ptr() for o in out), workspace, capi.cur_stream())
        rc = call(None, 0)
        ctx.sync_check()
        if (sentences, beams, V) == (2, 4, 5000):
            assert rc == 0
        else:
            assert rc == capi.EXB_ERR_NOMEM and (out == 7).all()
            room = 8 * sentences * beams * 5
            workspace = torch.full((room,), 255, device="cuda", dtype=torch.uint8)
            assert call(workspace.data_ptr(), room - 1) == capi.EXB_ERR_BAD_ARG
            assert call(workspace.data_ptr(), room) == 0
        ctx.sync_check()
        got = capi.beam_select(ctx, logits, scores, 4)
        ctx.sync_check()
        assert torch.equal(out[0].view(torch.float32), got[0]) and torch.equal(out[1], got[1]) and torch.equal(out[2], got[2])
        _check(got, _ref_scores(logits, scores, None, 0, 1.0), logits, 1.0, 4)


def test_a_row_of_sentences_longer_than_a_launch(ctx):
    """More sentences than one launch of the reordering has, and lengths that differ between them."""
    torch, capi = _mods()
    B = 700
    state = torch.randn((B * 2, 3, 5, 8), device="cuda", generator=_gen(1)).half()
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda").repeat(B, 1).contiguous()
    parents[::3] = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    lengths = (torch.arange(B, device="cuda") % 7).int()
    want = _ref_reorder(state, parents, lengths)
    capi.reorder_beams(ctx, state, parents, lengths)
    ctx.sync_check()
    assert torch.equal(state, want) and not math.isnan(float(state.sum()))
