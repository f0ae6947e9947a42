"""The operators behind a decoder where they can go wrong at the ends: values that are no numbers, masks and huge logits in the log
probabilities, large logits on the way to them, scales at fp32's ends and wide vocabularies in the product, results that lie over inputs,
another device."""
import math

import pytest

from tests.test_gpu_decoder_ops import DTYPES, _check_logprobs, _check_product, _gen, _masked_rows, _mods, _ref_logprobs, _rows

pytestmark = pytest.mark.gpu


def _tokens(torch, rows, V, given, g):
    return torch.randint(0, V, (rows, given), device="cuda", generator=g).int()


# ---- token log probabilities ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,V", [(8, 1), (8, 2), (8, 32), (8, 200), (8, 1000), (8, 5001), (8, 40000), (2, 131072), (1800, 2500), (400, 12001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_with_a_nan_at_the_first_token(ctx, rows, V, dtype):
    """NaN sorts above plus infinity and equal ones by their index, the first token's too; as many tokens as there are may be asked for."""
    torch, capi = _mods()
    g = _gen(rows + V)
    x = (torch.randn((rows, V), device="cuda", generator=g) * 3).to(getattr(torch, dtype))
    x[0::8, 0] = math.nan
    x[1::8] = math.nan
    x[2::8, 0] = -math.nan
    x[2::8, V - 1] = math.nan
    x[3::8] = -math.inf
    x[3::8, 0] = math.nan
    x[4::8, 0] = math.inf
    x[5::8, V // 2] = math.nan
    x[6::8] = -math.inf
    x[6::8, V - 1] = -math.nan
    tokens = _tokens(torch, rows, V, 2, g)
    for top in sorted({1, min(V, 5), min(V, 32)}):
        for pad, offset in ((0, 0), (1, 1)):
            _check_logprobs(ctx, _rows(x, pad, offset), tokens, top, 0.7)

@pytest.mark.parametrize("rows,V", [(6, 900), (6, 40000), (2, 131072), (1800, 2500), (400, 12001)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_token_logprobs_of_a_huge_logit_behind_others(ctx, rows, V, dtype):
    """A thread that has added up small logits meets one near the type's end: its row's other tokens are nothing, and the entropy is 0."""
    torch, capi = _mods()
    x = torch.zeros((rows, V), device="cuda", dtype=getattr(torch, dtype))
    at = torch.arange(rows, device="cuda") * 997 % (V // 3) + V * 2 // 3
    x[torch.arange(rows, device="cuda"), at] = 2.0 ** 123      # (exact times log2 e, so that the one pass answers it)
    tokens = torch.stack([at, at * 0], 1).int()
    for scale in (0.5, 1.0, 2.0):
        _check_logprobs(ctx, x, tokens, 3, scale)

@pytest.mark.parametrize("rows,V", [(3, 900), (3, 40000), (2, 131072), (1800, 2500), (400, 12001)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_token_logprobs_of_logits_further_apart_than_fp32_reaches(ctx, rows, V, dtype):
    """Distances that are no fp32 number any more at a large scale: those tokens are nothing, and the entropy is 0, not NaN."""
    torch, capi = _mods()
    x = torch.full((rows, V), torch.finfo(getattr(torch, dtype)).min, device="cuda", dtype=getattr(torch, dtype))
    x[1::2] = -9e29
    x[:, V // 2] = 2.0 ** 101
    tokens = torch.tensor([[V // 2, 0]], device="cuda").repeat(rows, 1).int()
    _check_logprobs(ctx, x, tokens, 3, 9e7)

@pytest.mark.parametrize("rows,V", [(3, 900), (1800, 2500), (3, 40000), (2, 131072), (400, 20001)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_masked_with_low_values_take_the_same_way(ctx, rows, V, dtype):
    """Masks of the type's lowest value, or of one that is low enough, are answered by the same sums in the same order as minus infinity,
    whatever the scale and however many of a thread's tokens are masked: equal bits."""
    torch, capi = _mods()
    t = getattr(torch, dtype)
    g = _gen(V)
    x = (torch.randn((rows, V), device="cuda", generator=g) * 4).to(t)
    mask = torch.rand((rows, V), device="cuda", generator=g) < 0.6
    mask[:, V // 5: V * 3 // 5] = True
    mask[1:, : V // 5] = True
    tokens = torch.arange(V - 3, V, device="cuda").repeat(rows, 1).int()
    mask[:, V - 3:] = False
    want = {s: capi.token_logprobs(ctx, x.masked_fill(mask, -math.inf), tokens, top=5, scale=s) for s in (0.3, 0.5, 1.0, 1.5)}
    for low in (torch.finfo(t).min,) + (() if dtype == "float16" else (-2e30, -1e38)):
        for scale, w in want.items():
            got = capi.token_logprobs(ctx, x.masked_fill(mask, low), tokens, top=5, scale=scale)
            ctx.sync_check()
            assert all(torch.equal(a, b) for a, b in zip(got, w)), (low, scale)
    _check_logprobs(ctx, x.masked_fill(mask, torch.finfo(t).min), tokens, 5, 0.5)

@pytest.mark.parametrize("rows,V", [(2000, 40), (64, 1000), (1800, 2500), (100, 40000), (16, 131072)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_stay_in_their_range(ctx, rows, V, dtype):
    """No log probability above 0 and no entropy below it, in rows of which a mask leaves one token, or of which one has nearly everything."""
    torch, capi = _mods()
    g = _gen(V)
    at = torch.randint(0, V, (rows, 1), device="cuda", generator=g)
    own = torch.randn((rows, 1), device="cuda", generator=g) * 10
    for others in (torch.full((rows, V), -math.inf, device="cuda"), torch.randn((rows, V), device="cuda", generator=g) - 60):
        x = others.scatter(1, at, own).to(getattr(torch, dtype))
        for scale in (0.7, 1.0, 1.3):
            lp, entropy, best, tokens = capi.token_logprobs(ctx, x, at.int(), top=1, scale=scale)
            ctx.sync_check()
            assert (lp <= 0).all() and (best <= 0).all() and (entropy >= 0).all()
            assert torch.equal(tokens, at.int())
        _check_logprobs(ctx, x, at.int(), 2, 1.3)

@pytest.mark.parametrize("V", [129, 200, 256, 262])
def test_token_logprobs_of_short_rows_with_many_alternatives(ctx, V):
    """Rows of so few tokens that not every lane of a warp holds some, and as many alternatives as lanes that do or more: answered in one
    go like others, where a pass over the row for each alternative took ten times as long."""
    torch, capi = _mods()
    rows = 8192
    x = torch.randn((rows, V), device="cuda", generator=_gen(V)).half()
    tokens = torch.zeros((rows, 1), device="cuda", dtype=torch.int32)
    _check_logprobs(ctx, x, tokens, 32, 1.0)

    def least(top):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                capi.token_logprobs(ctx, x, tokens, top=top)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    assert least(32) < 4 * least(10)


@pytest.mark.parametrize("V", [130, 200, 262, 500, 600])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_of_short_rows_with_masks_and_many_alternatives(ctx, V, dtype):
    """Equal logits among more candidates than are put in order at once: the lower indexes come first."""
    torch, capi = _mods()
    g = _gen(V)
    x = _masked_rows(torch, V, getattr(torch, dtype), g)
    x[11] = torch.randint(0, 3, (V,), device="cuda", generator=g)
    x[12, 1::2] = 0.5
    tokens = _tokens(torch, 16, V, 2, g)
    for top in (15, 24, 32):
        for pad, offset in ((0, 0), (1, 1)):
            _check_logprobs(ctx, _rows(x, pad, offset), tokens, top, 0.9)


# ---- the product ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M", [1, 2, 16, 17, 64])
def test_fp8_matmul_of_few_rows_with_extreme_scales(ctx, M):
    """Scales that span the range of fp32 between blocks, and zero blocks, with nothing infinite: every row is right."""
    torch, capi = _mods()
    g = _gen(M)
    N, K = 300, 640
    x = torch.randn((M, K), device="cuda", generator=g)
    v = torch.randn((N, K), device="cuda", generator=g)
    x[:, :128] *= 1e18
    x[:, 128:256] *= 1e-18
    x[:, 256:384] = 0
    v[:, :128] *= 1e-18
    v[:, 128:256] *= 1e18
    a, sa = capi.quantize_blocks(ctx, x)
    w, sw = capi.quantize_blocks(ctx, v, 128)
    y = capi.fp8_matmul(ctx, a, sa, w, sw, None, capi.EXB_F32)
    ctx.sync_check()
    _check_product(y, a, sa, w, sw, None, "float32")


@pytest.mark.parametrize("M,N,K", [(1, 128256, 300), (16, 70001, 260), (64, 131072, 128), (70, 66000, 200), (300, 131071, 150)])
def test_fp8_matmul_with_a_vocabulary(ctx, M, N, K):
    torch, capi = _mods()
    g = _gen(N)
    a, sa = capi.quantize_blocks(ctx, torch.randn((M, K), device="cuda", generator=g).half())
    w, sw = capi.quantize_blocks(ctx, torch.randn((N, K), device="cuda", generator=g).half() * 0.05, 128)
    for dtype in ("float32", "bfloat16"):
        y = capi.fp8_matmul(ctx, a, sa, w, sw, None, capi.exb_dtype_of(getattr(torch, dtype)))
        ctx.sync_check()
        _check_product(y, a, sa, w, sw, None, dtype)


# ---- together ------------------------------------------------------------------------------------------------------------

def test_token_head_keeps_logits_in_fp32(ctx):
    """Log probabilities are as good as their logits: unless told otherwise these are fp32, where fp16 would end at 65504."""
    torch, capi = _mods()
    from excalibur_b200.token_head import TokenHead
    g = _gen(11)
    C, V = 256, 500
    head = TokenHead(ctx, torch.randn((V, C), device="cuda", generator=g) * 1e4, torch.ones(C, device="cuda"))
    h, x = torch.randn((4, C), device="cuda", generator=g), torch.zeros((4, C), device="cuda")
    _, logits = head.logits(h, x)
    assert logits.dtype == torch.float32 and float(logits.abs().max()) > 65504
    given, entropy, best, tokens = head.scores(h, x, torch.zeros((4, 1), device="cuda", dtype=torch.int32), top=3, temperature=1e4)
    ctx.sync_check()
    assert all(torch.isfinite(v).all() for v in (given, entropy, best))
    assert torch.equal(tokens, _ref_logprobs(logits, torch.zeros((4, 1), device="cuda", dtype=torch.int32), 3, 1e-4)[3])


# ---- results over inputs -------------------------------------------------------------------------------------------------

def _refused(capi, calls):
    for i, call in enumerate(calls):
        with pytest.raises(capi.ExbError) as e:
            call()
        assert e.value.code == capi.EXB_ERR_BAD_ARG, i


def test_residual_norm_refuses_results_over_inputs(ctx):
    """A result may take h's or x's own place; over any other part of an input, or over another result, some rows would be read after
    they were written."""
    torch, capi = _mods()
    C = 256
    w = torch.ones(C, device="cuda")
    buf = torch.randn((12, C), device="cuda")
    h, x, wide = torch.randn((8, C), device="cuda"), buf[:8], torch.randn((8, 4 * C), device="cuda")
    flat = buf.view(-1)
    as_bytes = buf.view(torch.float8_e4m3fn)
    _refused(capi, [
        lambda: capi.residual_norm(ctx, h, x, gate=x[3:4], weight=w, r=x),
        lambda: capi.residual_norm(ctx, h, x, gate=x[2:6], gate_rows=2, weight=w, r=x),
        lambda: capi.residual_norm(ctx, h, x, gate=x[7:8], weight=w, n=x),
        lambda: capi.residual_norm(ctx, h, x, r=buf[1:9]),
        lambda: capi.residual_norm(ctx, h, x, r=buf[4:12]),
        lambda: capi.residual_norm(ctx, x, h, weight=w, n=buf[2:10]),
        lambda: capi.residual_norm(ctx, h, x, r=flat[1:1 + 8 * C].view(8, C)),
        lambda: capi.residual_norm(ctx, h, x, r=buf.as_strided((8, C), (C + 8, 1))),
        lambda: capi.residual_norm(ctx, h, x, weight=w, r=wide[:, :C], n=wide[:, C // 2: C // 2 + C]),
        lambda: capi.residual_norm(ctx, h, x, weight=w, r=wide.view(-1)[:8 * C].view(8, C), n=wide[:, C:2 * C]),
        lambda: capi.residual_norm(ctx, wide[:, :C], wide[:, C:2 * C], r=wide[:, C - 8:2 * C - 8]),
        lambda: capi.residual_norm(ctx, wide[:, :C], h, r=wide.as_strided((8, C), (4 * C - 8, 1), 3 * C + 8)),
        lambda: capi.residual_norm(ctx, h, x, weight=x[0], r=x),
        lambda: capi.residual_norm(ctx, h, x, post_weight=x[7], weight=w, n=x),
        lambda: capi.residual_norm(ctx, h, x, weight=w, quantized=True, n=as_bytes[:8, :C]),
        lambda: capi.residual_norm(ctx, h, x, weight=w, quantized=True, r=wide[:, :C], n=wide.view(torch.float8_e4m3fn)[:, C:2 * C]),
    ])
    ctx.sync_check()


def test_residual_norm_takes_columns_of_a_wider_matrix(ctx):
    """Inputs and results that lie next to each other in the rows of one matrix share no element, and h's and x's own places stay open."""
    torch, capi = _mods()
    g = _gen(21)
    for C in (256, 250):
        w = torch.rand(C, device="cuda", generator=g)
        h, x, gate = (torch.randn((9, C), device="cuda", generator=g) for _ in range(3))
        want = capi.residual_norm(ctx, h, x, gate=gate, gate_rows=1, weight=w)
        wide = torch.zeros((9, 5 * C), device="cuda")
        parts = [wide[:, i * C:(i + 1) * C] for i in range(5)]
        for v, p in zip((h, x, gate), parts):
            p.copy_(v)
        r, n = capi.residual_norm(ctx, parts[0], parts[1], gate=parts[2], gate_rows=1, weight=w, r=parts[3], n=parts[4])
        ctx.sync_check()
        assert torch.equal(r, want[0]) and torch.equal(n, want[1]) and torch.equal(parts[0], h) and torch.equal(parts[2], gate)
        r, n = capi.residual_norm(ctx, parts[0], parts[1], gate=parts[2], gate_rows=1, weight=w, r=parts[1], n=parts[0])
        ctx.sync_check()
        assert torch.equal(r, want[0]) and torch.equal(n, want[1]) and torch.equal(parts[2], gate)
        # one row: its distance to the next does not matter
        one = torch.stack([h[0], x[0], torch.zeros_like(x[0])])
        r, _ = capi.residual_norm(ctx, one[0:1], one[1:2], r=one[2:3])
        r2, _ = capi.residual_norm(ctx, h[:1], x[:1])
        ctx.sync_check()
        assert torch.equal(r, r2)
        both = x[:1].clone()
        capi.residual_norm(ctx, h[:1], both, r=both)
        ctx.sync_check()
        assert torch.equal(both, r2)
        # x and h the same
        same = h.clone()
        capi.residual_norm(ctx, same, same, r=same)
        r3, _ = capi.residual_norm(ctx, h, h)
        ctx.sync_check()
        assert torch.equal(same, r3)


def test_other_results_over_inputs_are_refused(ctx):
    torch, capi = _mods()
    x = torch.randn((8, 256), device="cuda")
    as_bytes, floats = x.view(torch.float8_e4m3fn), torch.zeros(4096, device="cuda")
    _refused(capi, [
        lambda: capi.quantize_blocks(ctx, x, q=as_bytes[:, :256]),
        lambda: capi.quantize_blocks(ctx, x, q=as_bytes[:, 512:768]),
        lambda: capi.quantize_blocks(ctx, x, 128, q=as_bytes[:, 768:1024]),
        lambda: capi.quantize_blocks(ctx, x, scales=x[:2, :8]),
        lambda: capi.quantize_blocks(ctx, x, q=floats[:512].view(torch.float8_e4m3fn).view(8, 256), scales=floats[500:516].view(2, 8)),
    ])
    # 8 bits between the columns of a wider matrix share nothing with them
    wide = torch.zeros((8, 1024), device="cuda")
    wide[:, :256] = x
    q, s = capi.quantize_blocks(ctx, wide[:, :256], q=wide.view(torch.float8_e4m3fn)[:, 2048:2304], scales=wide[:2, 300:308])
    want_q, want_s = capi.quantize_blocks(ctx, x)
    ctx.sync_check()
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s, want_s) and torch.equal(wide[:, :256], x)

    w, sw = capi.quantize_blocks(ctx, x, 128)
    a, sa = want_q, want_s
    bias = torch.zeros(8, device="cuda")
    half = capi.EXB_F16
    L, st, addr = capi.lib(), None, lambda t: t.data_ptr()  # noqa: E731

    def matmul(y_at, ys=8):
        d = capi.MatmulDesc(M=8, N=8, K=256, y_dtype=half, a_stride=256, a_scale_stride=8, w_stride=256, w_scale_stride=2, y_stride=ys)
        import ctypes
        return L.exb_fp8_matmul_fwd(ctx.handle, ctypes.byref(d), addr(a), addr(sa), addr(w), addr(sw), addr(bias), y_at, st)
    for at in (addr(a), addr(a) + 8 * 256 - 16, addr(w) + 512, addr(sa) + 32, addr(sw), addr(bias) + 16):
        assert matmul(at) == capi.EXB_ERR_BAD_ARG

    logits, tokens = torch.randn((4, 64), device="cuda"), torch.zeros((4, 2), device="cuda", dtype=torch.int32)
    out = torch.zeros(256, device="cuda")

    def scores(lp=addr(out), entropy=addr(out) + 64, top_lp=addr(out) + 128, top_tokens=addr(out) + 256):
        import ctypes
        d = capi.LogprobsDesc(rows=4, stride=64, V=64, dtype=capi.EXB_F32, n_given=2, top=3, scale=1.0)
        return L.exb_token_logprobs_fwd(ctx.handle, ctypes.byref(d), addr(logits), addr(tokens), lp, entropy, top_lp, top_tokens, st)
    assert scores() == capi.EXB_OK
    for k in (dict(lp=addr(logits)), dict(lp=addr(tokens)), dict(entropy=addr(logits) + 4 * 255), dict(top_lp=addr(tokens) + 28), dict(top_tokens=addr(logits) + 100),
              dict(entropy=addr(out) + 28), dict(top_lp=addr(out) + 76), dict(top_tokens=addr(out) + 172), dict(lp=addr(out) + 256 + 44)):
        assert scores(**k) == capi.EXB_ERR_BAD_ARG, k
    ctx.sync_check()


# ---- another device ------------------------------------------------------------------------------------------------------

def test_a_context_of_another_device_than_the_current_one_is_refused(ctx):
    """A launch goes to the calling thread's current device, whatever the context's and the tensors': these have to be the same."""
    import ctypes as C
    torch, capi = _mods()
    # the context as it would be on the next device: its first field is the device
    other = (C.c_int32 * 10).from_buffer_copy((C.c_int32 * 10).from_address(C.cast(ctx.handle, C.c_void_p).value))
    assert other[0] == ctx.device == torch.cuda.current_device()
    other[0] += 1
    x = torch.randn((8, 256), device="cuda")
    q, s = capi.quantize_blocks(ctx, x)
    w, sw = capi.quantize_blocks(ctx, x, 128)
    out, L = torch.zeros_like(x), capi.lib()
    blocks = capi.BlocksDesc(rows=8, C=256, in_dtype=capi.EXB_F32, block_rows=1, x_stride=256, q_stride=256, scale_stride=8)
    matmul = capi.MatmulDesc(M=8, N=8, K=256, y_dtype=capi.EXB_F16, a_stride=256, a_scale_stride=8, w_stride=256, w_scale_stride=2, y_stride=8)
    norm = capi.NormDesc(rows=8, C=256, dtype=capi.EXB_F32, out_dtype=capi.EXB_F32, kind=0, eps=1e-5, residual_scale=1.0, h_stride=256, r_stride=256)
    scores = capi.LogprobsDesc(rows=8, stride=256, V=256, dtype=capi.EXB_F32, n_given=0, top=0, scale=1.0)
    X, Q, S, W, SW, Y = (t.data_ptr() for t in (x, q, s, w, sw, out))
    for handle, want in ((C.byref(other), capi.EXB_ERR_BAD_ARG), (ctx.handle, capi.EXB_OK)):
        assert L.exb_quantize_blocks_fwd(handle, C.byref(blocks), X, Q, S, None) == want
        assert L.exb_fp8_matmul_fwd(handle, C.byref(matmul), Q, S, W, SW, None, Y, None) == want
        assert L.exb_residual_norm_fwd(handle, C.byref(norm), X, None, None, None, None, None, None, Y, None, None, None) == want
        assert L.exb_token_logprobs_fwd(handle, C.byref(scores), X, None, None, Y, None, None, None) == want
        if want != capi.EXB_OK:
            assert "current device" in capi.last_error()
    ctx.sync_check()
