"""The operators behind a decoder (norms around a block, 8-bit blocks, their product, token log probabilities) against plain
implementations in 64 bits, at the sizes, strides, types and masks where they can go wrong."""
import math

import pytest

pytestmark = pytest.mark.gpu

DTYPES = ("float16", "bfloat16", "float32")
# half a unit in the last place, relative
ROUND = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
SMALLEST_HALF = 2.0 ** -25      # half the smallest fp16 number


def _mods():
    import torch
    from excalibur_b200 import capi
    return torch, capi


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(t, pad=0, offset=0):
    """The same matrix in rows that are pad elements further apart and start offset elements into their buffer."""
    import torch
    if not pad and not offset:
        return t
    buf = torch.full((t.shape[0] * (t.shape[1] + pad) + offset,), 7, device=t.device, dtype=t.dtype)
    v = buf[offset:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


# ---- blocks of e4m3 ------------------------------------------------------------------------------------------------------

def _blocked(x, block_rows):
    import torch
    rows, C = x.shape
    nr, nc = -(-rows // block_rows), -(-C // 128)
    wide = torch.zeros((nr * block_rows, nc * 128), dtype=x.dtype, device=x.device)
    wide[:rows, :C] = x
    return wide.view(nr, block_rows, nc, 128)


def _ref_quantized(x, block_rows):
    """The definition in IEEE fp32: the kernels have to give the same bits."""
    import torch
    rows, C = x.shape
    b = _blocked(x.float().cpu(), block_rows)
    amax = torch.nan_to_num(b.abs(), nan=0.0, posinf=math.inf).amax((1, 3), keepdim=True)
    scale = torch.maximum(amax / torch.tensor(448.0), torch.tensor(2.0 ** -126))
    v = b * (torch.tensor(1.0) / scale)
    q = v.clamp(-448, 448).to(torch.float8_e4m3fn).reshape(b.shape[0] * block_rows, -1)[:rows, :C]
    scale = scale[:, 0, :, 0]
    return q, scale.t().contiguous() if block_rows == 1 else scale


def _same_bits(q, ref):
    import torch
    a, b = q.cpu().float(), ref.float()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("rows,C", [(1, 1), (1, 127), (3, 128), (5, 129), (64, 4096), (33, 1000), (130, 257), (257, 136), (1, 16384), (129, 384)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_blocks(ctx, rows, C, dtype, block_rows):
    torch, capi = _mods()
    x = (torch.randn((rows, C), device="cuda", generator=_gen(rows * 7 + C)) * 3).to(getattr(torch, dtype))
    x[:, C // 2] *= 100
    for pad, offset in ((0, 0), (3, 1), (16, 8)):
        q, s = capi.quantize_blocks(ctx, _rows(x, pad, offset), block_rows)
        ctx.sync_check()
        rq, rs = _ref_quantized(x, block_rows)
        assert torch.equal(s.cpu(), rs)
        assert _same_bits(q, rq)
    # against 64 bits: half a step of a number with 4 significant bits, or of the block's smallest step (2^-9 of its scale)
    each = _blocked(torch.ones_like(x, dtype=torch.float64), block_rows) * (s.t() if block_rows == 1 else s).double()[:, None, :, None]
    each = each.reshape(-1, each.shape[2] * 128)[:rows, :C]
    v = x.double()
    assert ((q.double() * each - v).abs() <= (v.abs() * 2.0 ** -4 + each * 2.0 ** -10) * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("aligned", [True, False])
def test_quantize_blocks_at_the_ends_of_the_types(ctx, dtype, block_rows, aligned):
    torch, capi = _mods()
    t = getattr(torch, dtype)
    big, tiny = torch.finfo(t).max, torch.finfo(t).tiny
    x = torch.zeros((256, 512), device="cuda", dtype=t)
    x[0, 0:128] = big
    x[1, 0:128] = torch.linspace(-1, 1, 128, device="cuda") * (tiny if dtype == "float32" else 1e-7)
    x[2, 128] = math.inf
    x[2, 129] = 1
    x[3, 256] = math.nan
    x[3, 257] = 2
    x[4, 384] = -math.inf
    x[200, 3] = -0.0
    q, s = capi.quantize_blocks(ctx, x if aligned else _rows(x, 1, 1), block_rows)
    ctx.sync_check()
    rq, rs = _ref_quantized(x, block_rows)
    assert torch.equal(s.cpu(), rs) and _same_bits(q, rq)
    assert torch.isfinite(s[:, 1] if block_rows == 128 else s[:, 0]).any()
    if block_rows == 1:      # an infinity leaves no value in its block, a NaN only itself
        v = q.float() * s.t().repeat_interleave(128, 1)
        assert torch.isnan(v[2, 128:256]).all() and torch.isfinite(v[2, :128]).all()
        assert torch.isnan(v[3, 256]) and v[3, 257] == 2


def test_quantize_blocks_leaves_what_lies_between_rows(ctx):
    torch, capi = _mods()
    for C in (1, 100, 127, 129, 250):
        x = torch.randn((37, C), device="cuda", generator=_gen(C)).half()
        for br in (1, 128):
            wide = torch.full((37, 304), 0x55, device="cuda", dtype=torch.uint8)
            scales = torch.full((40, 64), -1.0, device="cuda")
            shape = (-(-C // 128), 37) if br == 1 else (1, -(-C // 128))
            capi.quantize_blocks(ctx, x, br, q=wide.view(torch.float8_e4m3fn)[:, :C], scales=scales[:shape[0], :shape[1]])
            ctx.sync_check()
            assert (wide[:, C:] == 0x55).all()
            assert (scales[:shape[0], :shape[1]] > 0).all() and (scales[shape[0]:] == -1).all() and (scales[:, shape[1]:] == -1).all()


# ---- the product ---------------------------------------------------------------------------------------------------------

def _dequantized(q, s, block_rows):
    v = q.double()
    s = s.double()
    if block_rows == 1:
        return v * s.t().repeat_interleave(128, 1)[:, :v.shape[1]]
    return v * s.repeat_interleave(128, 0)[:v.shape[0]].repeat_interleave(128, 1)[:, :v.shape[1]]


def _check_product(y, a, sa, w, sw, bias, dtype):
    """Sums of 128 products and of the blocks: each addition is off by a unit in fp32's last place (2^-23) at most of what has been added in
    magnitude; then the rounding to the result's type."""
    import torch
    A, W = _dequantized(a, sa, 1), _dequantized(w, sw, 128)
    ref, mag = A @ W.t(), A.abs() @ W.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    blocks = -(-a.shape[1] // 128)
    tol = (128 + blocks + 8) * 2.0 ** -23 * mag + ROUND[dtype] * ref.abs() + (SMALLEST_HALF if dtype == "float16" else 0)
    assert y.shape == ref.shape and torch.isfinite(y).all()
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 128, 128), (1, 4096, 4096), (1, 1000, 1234), (2, 257, 129), (5, 64, 16), (7, 130, 4096), (16, 512, 640), (17, 1000, 384), (31, 384, 2000),
    (33, 129, 300), (48, 2048, 1024), (64, 4096, 512), (65, 300, 1000), (100, 1408, 768), (128, 128, 128), (129, 129, 129), (200, 1000, 1111),
    (256, 256, 256), (257, 511, 400), (333, 1000, 1234), (512, 1024, 2048), (700, 2500, 200), (1000, 777, 999), (2048, 2048, 1024), (1500, 4000, 500),
    (4100, 300, 260), (300, 9000, 140)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_fp8_matmul(ctx, M, N, K, dtype):
    torch, capi = _mods()
    g = _gen(M * 31 + N * 7 + K)
    a, sa = capi.quantize_blocks(ctx, torch.randn((M, K), device="cuda", generator=g).half())
    w, sw = capi.quantize_blocks(ctx, torch.randn((N, K), device="cuda", generator=g).half() * 0.05, 128)
    bias = torch.randn(N, device="cuda", generator=g) if (M + N) % 2 else None
    dt = capi.exb_dtype_of(torch.empty(0, dtype=getattr(torch, dtype)))
    y = capi.fp8_matmul(ctx, a, sa, w, sw, bias, dt)
    again = capi.fp8_matmul(ctx, a, sa, w, sw, bias, dt)
    ctx.sync_check()
    _check_product(y, a, sa, w, sw, bias, dtype)
    assert torch.equal(y, again)


@pytest.mark.parametrize("M,N,K,dtype", [
    (1, 130, 1290, "float32"),      # parts of K that divide neither it nor the rows: 5 of 11 blocks,
    (9, 130, 1750, "bfloat16"),     # 7 of 14,
    (16, 4300, 1800, "float16"),    # 7, where each CTA gets 3 columns of 6 others at most,
    (15, 4900, 1540, "float32"),    # 6,
    (33, 6100, 1300, "float16"),    # 5,
    (50, 9001, 777, "bfloat16"),    # 3,
    (131, 2400, 800, "float32"),    # 3 of tiles of 128 columns,
    (100, 2500, 1700, "float16"),   # 6
])
def test_fp8_matmul_in_uneven_parts(ctx, M, N, K, dtype):
    test_fp8_matmul(ctx, M, N, K, dtype)


@pytest.mark.parametrize("M,N,K", [(3, 200, 300), (70, 200, 300), (300, 700, 1000), (600, 1100, 300)])
def test_fp8_matmul_takes_strides_and_writes_nothing_else(ctx, M, N, K):
    torch, capi = _mods()
    g = _gen(5)
    pitch = (K + 15) // 16 * 16 + 32
    # what lies between the rows are NaN: reading any of it shows
    wide_a = torch.full((M, pitch), 0x7F, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    wide_w = torch.full((N, pitch), 0x7F, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    blocks = -(-K // 128)
    wide_sa = torch.full((blocks, M + 5), math.nan, device="cuda")
    wide_sw = torch.full((-(-N // 128), blocks + 3), math.nan, device="cuda")
    a, sa = capi.quantize_blocks(ctx, torch.randn((M, K), device="cuda", generator=g), q=wide_a[:, :K], scales=wide_sa[:, :M])
    w, sw = capi.quantize_blocks(ctx, torch.randn((N, K), device="cuda", generator=g), 128, q=wide_w[:, :K], scales=wide_sw[:, :blocks])
    for dtype in DTYPES:
        for offset, pad in ((0, 8), (1, 3)):
            buf = torch.full((M * (N + pad) + offset,), 77, device="cuda", dtype=getattr(torch, dtype))
            wide = buf[offset:].view(M, N + pad)
            y = capi.fp8_matmul(ctx, a, sa, w, sw, None, capi.exb_dtype_of(buf), y=wide[:, :N])
            ctx.sync_check()
            _check_product(y, a, sa, w, sw, None, dtype)
            assert (wide[:, N:] == 77).all() and (buf[:offset] == 77).all()


@pytest.mark.parametrize("M", [1, 40, 200, 600])
def test_fp8_matmul_with_extreme_scales(ctx, M):
    """Scales that span the range of fp32 between blocks, zero blocks, and rows that hold an infinity: only those are NaN."""
    torch, capi = _mods()
    g = _gen(M)
    N, K = 300, 640
    x = torch.randn((M, K), device="cuda", generator=g)
    x[:, :128] *= 1e18
    x[:, 128:256] *= 1e-18
    x[:, 256:384] = 0
    x[M // 2, 400] = math.inf
    v = torch.randn((N, K), device="cuda", generator=g)
    v[:, :128] *= 1e-18
    v[:, 128:256] *= 1e18
    a, sa = capi.quantize_blocks(ctx, x)
    w, sw = capi.quantize_blocks(ctx, v, 128)
    y = capi.fp8_matmul(ctx, a, sa, w, sw, None, capi.EXB_F32)
    ctx.sync_check()
    assert torch.isnan(y[M // 2]).all()
    keep = [i for i in range(M) if i != M // 2]
    if keep:
        _check_product(y[keep], a[keep], sa[:, keep], w, sw, None, "float32")


@pytest.mark.parametrize("quantized", [False, True])
def test_residual_norm_refuses_the_gate_as_a_result(ctx, quantized):
    """A gate that several rows share would be read by one row after another has written it."""
    torch, capi = _mods()
    h = torch.randn((4, 256), device="cuda").half()
    gate = torch.randn((4, 256), device="cuda").half()
    w = torch.ones(256, device="cuda")
    with pytest.raises(capi.ExbError):
        capi.residual_norm(ctx, h, gate=gate, weight=w, quantized=quantized, r=gate)
    if not quantized:
        with pytest.raises(capi.ExbError):
            capi.residual_norm(ctx, h, gate=gate, weight=w, n=gate)
    ctx.sync_check()


def test_fp8_matmul_on_another_stream_and_in_a_graph(ctx):
    torch, capi = _mods()
    g = _gen(9)
    a, sa = capi.quantize_blocks(ctx, torch.randn((33, 500), device="cuda", generator=g))
    w, sw = capi.quantize_blocks(ctx, torch.randn((270, 500), device="cuda", generator=g), 128)
    want = capi.fp8_matmul(ctx, a, sa, w, sw)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = capi.fp8_matmul(ctx, a, sa, w, sw)
        ctx.sync_check()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.fp8_matmul(ctx, a, sa, w, sw, y=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        ctx.sync_check()
        assert torch.equal(out, want)


# ---- norms around a block ------------------------------------------------------------------------------------------------

def _ref_norm(v, kind, weight, bias, eps):
    """(norm, its spread's reciprocal root, what the mean took part in)"""
    mean = v.mean(1, keepdim=True) if kind else v.new_zeros((v.shape[0], 1))
    k = ((v - mean) ** 2).mean(1, keepdim=True).add(eps).rsqrt()
    n = (v - mean) * k * weight.double()
    return (n if bias is None else n + bias.double()), k, mean.abs()


def _ref_residual(h, x, post, post_bias, gate, gate_rows, scale, weight, bias, kind, eps):
    import torch
    u = h.double()
    mag = u.abs()
    if post is not None:
        n, k, mean = _ref_norm(u, kind, post, post_bias, eps)
        mag = (mag + mean) * k * post.double().abs() + n.abs() + (0 if post_bias is None else post_bias.double().abs())
        u = n
    if gate is not None:
        at = torch.arange(h.shape[0], device=h.device) // gate_rows if gate_rows else torch.zeros(h.shape[0], device=h.device, dtype=torch.long)
        g = gate.double()[at]
        u, mag = u * g, mag * g.abs()
    u, mag = u * scale, mag * abs(scale)
    if x is not None:
        u, mag = u + x.double(), mag + x.double().abs()
    n, n_mag = None, None
    if weight is not None:
        n, k, mean = _ref_norm(u, kind, weight, bias, eps)
        # what a row's sum is off by reaches every element through the norm and the mean
        n_mag = (mag + mean) * k * weight.double().abs() + n.abs() + (0 if bias is None else bias.double().abs())
        if kind:
            n_mag = n_mag + mag.mean(1, keepdim=True) * k * weight.double().abs()
    return u, mag, n, n_mag


# fp32 sums of up to 64 values in a row and a tree above them: 74 additions, half of which the square root keeps, and a
# dozen roundings more, of half a unit each
SUMS = (74 + 12) * 2.0 ** -24


def _check_norm(got, ref, mag, dtype, what):
    tol = 3 * SUMS * mag + ROUND[dtype] * ref.abs() + (SMALLEST_HALF if dtype == "float16" else 0)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (what, float((err / tol).max()))


@pytest.mark.parametrize("rows,C", [(1, 1), (1, 8), (3, 7), (1, 4096), (2, 255), (5, 256), (700, 64), (700, 300), (700, 512), (350, 1000), (320, 1030), (9, 2048), (600, 2048),
                                    (3, 8192), (400, 4104), (7, 8200), (301, 8193), (2, 16384), (2, 16392), (3, 32768), (2, 32767)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [0, 1])
def test_residual_norm(ctx, rows, C, dtype, kind):
    torch, capi = _mods()
    t = getattr(torch, dtype)
    g = _gen(rows + C * 3 + kind)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    h, x = rand(rows, C).to(t), rand(rows, C).to(t)
    w, b, pw, pb = 1 + 0.1 * rand(C), 0.1 * rand(C), 1 + 0.1 * rand(C), 0.1 * rand(C)
    for post, gate_rows, layout, with_x in ((False, None, (0, 0), True), (True, 0, (0, 0), True), (True, 1, (8, 8), True), (False, 3, (1, 1), True), (True, None, (0, 0), False)):
        gate = None if gate_rows is None else rand(1 if gate_rows == 0 else -(-rows // gate_rows), C).to(t)
        args = dict(post_weight=pw if post else None, post_bias=pb if post and kind else None, gate=None if gate is None else _rows(gate, *layout),
                    gate_rows=gate_rows or 0, residual_scale=0.5, weight=w, bias=b if kind else None, kind=kind, eps=1e-3)
        xx = x if with_x else None
        r, n = capi.residual_norm(ctx, _rows(h, *layout), None if xx is None else _rows(xx, *layout), **args)
        r2, q, s = capi.residual_norm(ctx, _rows(h, *layout), None if xx is None else _rows(xx, *layout), quantized=True, **args)
        ctx.sync_check()
        ur, mag, un, n_mag = _ref_residual(h, xx, pw if post else None, pb if post and kind else None, gate, gate_rows or 0, 0.5, w, b if kind else None, kind, 1e-3)
        _check_norm(r, ur, mag, dtype, "r")
        _check_norm(n, un, n_mag, dtype, "n")
        assert torch.equal(r, r2)
        # the scale is the largest value's; each value half a step of e4m3 off at most
        v = _dequantized(q, s, 1)
        big = _blocked(un.abs(), 1)[:, 0].amax(2).t()
        off = _blocked(n_mag, 1)[:, 0].amax(2).t() * 3 * SUMS
        assert ((s.double() * 448 - big).abs() <= off + big * 2.0 ** -22 + 448 * 2.0 ** -126).all()
        each = s.double().t().repeat_interleave(128, 1)[:, :C]
        assert ((v - un).abs() <= (un.abs() * 2.0 ** -4 + each * 2.0 ** -10) * (1 + 2.0 ** -20) + 1.1 * 3 * SUMS * n_mag).all()


def test_residual_norm_in_place_and_one_output(ctx):
    torch, capi = _mods()
    g = _gen(3)
    for C in (96, 1000, 5000, 5001):
        h, x = torch.randn((70, C), device="cuda", generator=g).half(), torch.randn((70, C), device="cuda", generator=g).half()
        w = torch.rand(C, device="cuda", generator=g)
        r, n = capi.residual_norm(ctx, h, x, weight=w)
        for where in ("x", "h"):
            h2, x2 = h.clone(), x.clone()
            r_at, n_at = (x2, h2) if where == "x" else (h2, x2)
            r2, n2 = capi.residual_norm(ctx, h2, x2, weight=w, r=r_at, n=n_at)
            ctx.sync_check()
            assert torch.equal(r2, r) and torch.equal(n2, n) and r2.data_ptr() == r_at.data_ptr()
        only_r, none = capi.residual_norm(ctx, h, x)
        ctx.sync_check()
        assert none is None and torch.equal(only_r, r)


def test_residual_norm_of_zeros_and_values_that_are_no_numbers(ctx):
    torch, capi = _mods()
    h = torch.zeros((4, 300), device="cuda")
    x = torch.zeros((4, 300), device="cuda")
    x[1, 5] = math.nan
    x[2, 299] = math.inf
    w = torch.ones(300, device="cuda")
    for kind in (0, 1):
        r, n = capi.residual_norm(ctx, h, x, weight=w, kind=kind, eps=1e-5)
        ctx.sync_check()
        assert torch.equal(torch.nan_to_num(r, nan=-5.0), torch.nan_to_num(x, nan=-5.0))
        assert (n[0] == 0).all() and (n[3] == 0).all() and torch.isnan(n[1]).all()
        assert torch.isnan(n[2, 299]) and (kind or (n[2, :299] == 0).all())


# ---- token log probabilities ---------------------------------------------------------------------------------------------

def _ref_logprobs(logits, tokens, top, scale):
    import torch
    x = logits.double()
    V = x.shape[1]
    # (from the largest logit on: with masks of fp32's lowest value 64 bits do not hold lse either)
    z = (x - x.amax(1, keepdim=True)) * scale
    lse = torch.logsumexp(z, 1, keepdim=True)
    empty = (x == -math.inf).all(1, keepdim=True)
    bad = (torch.isnan(x) | (x == math.inf)).any(1, keepdim=True)
    lp = torch.where(empty, -math.inf, torch.where(bad, math.nan, z - lse))
    p = lp.exp()
    entropy = torch.where(bad[:, 0], math.nan, -torch.where(p > 0, p * lp, 0.0).sum(1))
    inside = (tokens >= 0) & (tokens < V)
    given = torch.where(inside, lp.gather(1, tokens.long().clamp(0, V - 1)), torch.where(tokens < 0, 0.0, math.nan).double())
    order = torch.sort(torch.where(torch.isnan(x), math.inf, x), dim=1, descending=True, stable=True).indices
    if torch.isnan(x).any():      # NaN stands above infinity
        order = torch.gather(order, 1, torch.sort(torch.isnan(x).gather(1, order).to(torch.int8), dim=1, descending=True, stable=True).indices)
    best = order[:, :top]
    return given, entropy, lp.gather(1, best), best.int()


def _check_logprobs(ctx, logits, tokens, top, scale):
    """A thread adds up to max(V / 512, 128) values one after the other and a tree of 30 joins them, half a unit each; the powers
    of two are off by 2^-22, and their arguments by a few half units."""
    torch, capi = _mods()
    lp, entropy, top_lp, top_tokens = capi.token_logprobs(ctx, logits, tokens, top=top, scale=scale)
    ctx.sync_check()
    rlp, rent, rtop, rbest = _ref_logprobs(logits, tokens, top, scale)
    V = logits.shape[1]
    tol = (max(V / 512, 128) + 30) * 2.0 ** -24 + 2.0 ** -21

    def near(got, ref, tol):
        got, ref = got.double(), ref.float().double()      # (a difference of two of fp32's ends is infinite in fp32)
        fine = torch.isfinite(ref)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
        err = (got - ref).abs()[fine]
        bound = (tol + 2.0 ** -21 * ref.abs())[fine]
        assert (err <= bound).all(), float((err / bound).max())
    near(lp, rlp, tol)
    near(entropy, rent, tol * (4 + math.log(V)))
    if top:
        assert torch.equal(top_tokens, rbest)
        near(top_lp, rtop, tol)


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 2), (3, 7), (2, 31), (5, 33), (300, 100), (256, 1000), (4, 1023), (3, 4096), (2, 4097), (600, 2050), (1, 50001), (5, 50001),
                                    (40, 32000), (160, 20001), (1, 131072), (2, 262147), (3, 9000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs(ctx, rows, V, dtype):
    torch, capi = _mods()
    g = _gen(rows * 13 + V)
    x = (torch.randn((rows, V), device="cuda", generator=g) * 3).to(getattr(torch, dtype))
    for given, top, scale, (pad, offset) in ((1, min(V, 20), 1.0, (0, 0)), (3, min(V, 5), 0.7, (8, 8)), (2, min(V, 32), 1.3, (1, 1)), (1, 0, 2.0, (0, 0)), (1, 1, 1.0, (5, 3))):
        tokens = torch.randint(0, V, (rows, given), device="cuda", generator=g).int()
        _check_logprobs(ctx, _rows(x, pad, offset), tokens, top, scale)


def _masked_rows(torch, V, t, g):
    """16 rows: masks that leave nothing, one or a few tokens, the type's lowest value, equal values, and values that are no numbers."""
    low = torch.finfo(t).min
    x = torch.randn((16, V), device="cuda", generator=g) * 4
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, V // 3] = 2.5
    x[2] = -math.inf
    x[2, 3::7] = torch.randn_like(x[2, 3::7])
    x[3] = low
    x[4] = low
    x[4, V - 1] = 1.0
    x[4, 5] = 1.0
    x[5] = 0.25
    x[6] = 0.0
    x[6, 1::2] = -0.0
    x[7, V // 2] = math.inf
    x[8, V - 2] = math.nan
    x[9] = -math.inf
    x[9, 1] = math.nan
    x[10] = torch.finfo(t).max
    x[11] = torch.arange(V, device="cuda") * (8.0 / V)
    x[12] = -torch.arange(V, device="cuda") * (8.0 / V)
    x[13, : V // 2] = -math.inf
    x[14] = -math.inf
    x[14, -1] = low
    x[15] = low
    x[15, 7] = torch.finfo(t).max
    return x.to(t)


@pytest.mark.parametrize("V", [40, 1000, 5001, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_with_masks(ctx, V, dtype):
    """Rows of which the mask leaves nothing, one or a few tokens, masks of the type's lowest value, rows of equal values, and values that are no numbers."""
    torch, capi = _mods()
    t = getattr(torch, dtype)
    g = _gen(V)
    x = _masked_rows(torch, V, t, g)
    tokens = torch.stack([torch.randint(0, V, (16,), device="cuda", generator=g), torch.full((16,), 5, device="cuda"), torch.full((16,), -1, device="cuda"),
                          torch.full((16,), V, device="cuda"), torch.full((16,), V // 3, device="cuda")], 1).int()
    for scale in (1.0, 2.0, 0.5):
        for top in (0, 1, 5, 20, 32):
            for pad, offset in ((0, 0), (1, 1)):
                _check_logprobs(ctx, _rows(x, pad, offset), tokens, top, scale)


@pytest.mark.parametrize("rows,V", [(1792, 500), (1792, 2500), (1792, 8000), (304, 12001), (80, 30000)])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_token_logprobs_with_masks_in_many_rows(ctx, rows, V, dtype):
    """The same rows often enough that a warp has one each (in 16 bits up to 8192 tokens), or a narrow CTA; between them rows without masks."""
    torch, capi = _mods()
    t = getattr(torch, dtype)
    g = _gen(rows + V)
    x = (torch.randn((rows, V), device="cuda", generator=g) * 4).to(t)
    x[::2] = _masked_rows(torch, V, t, g).repeat(-(-rows // 32), 1)[: (rows + 1) // 2]
    tokens = torch.randint(-1, V + 1, (rows, 2), device="cuda", generator=g).int()
    for top, scale, (pad, offset) in ((0, 1.0, (0, 0)), (5, 0.7, (1, 1)), (32, 1.3, (0, 0))):
        _check_logprobs(ctx, _rows(x, pad, offset), tokens, top, scale)


def test_token_logprobs_differences_in_huge_logits(ctx):
    """What counts is the distance to the largest logit, wherever that lies."""
    torch, capi = _mods()
    base = torch.randn((4, 3000), device="cuda", generator=_gen(1))
    for shift in (0.0, 1e4, -1e4, 3e6):
        x = base + shift
        _check_logprobs(ctx, x, torch.full((4, 1), 17, device="cuda", dtype=torch.int32), 10, 1.0)


def test_token_logprobs_past_32_bits(ctx):
    """Rows that lie more than 2^31 elements into the tensor."""
    torch, capi = _mods()
    V, apart = 1001, 1 << 26
    buf = torch.empty(40 * apart + V, device="cuda", dtype=torch.float16)
    x = buf.as_strided((41, V), (apart, 1))
    small = torch.randn((41, V), device="cuda", generator=_gen(2)).half()
    x.copy_(small)
    tokens = torch.arange(41, device="cuda", dtype=torch.int32)[:, None]
    for top in (0, 7):
        a = capi.token_logprobs(ctx, x, tokens, top=top)
        b = capi.token_logprobs(ctx, small, tokens, top=top)
        ctx.sync_check()
        # (rows at another alignment are added up in another order)
        assert torch.allclose(a[0], b[0], rtol=1e-5, atol=1e-5) and torch.allclose(a[1], b[1], rtol=1e-5, atol=1e-5)
        if top:
            assert torch.equal(a[3], b[3])


def test_same_results_every_time(ctx):
    torch, capi = _mods()
    g = _gen(4)
    x = torch.randn((3, 70001), device="cuda", generator=g).half()
    tokens = torch.zeros((3, 1), device="cuda", dtype=torch.int32)
    first = capi.token_logprobs(ctx, x, tokens, top=20)
    for _ in range(5):
        again = capi.token_logprobs(ctx, x, tokens, top=20)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    ctx.sync_check()


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_nothing_to_do(ctx):
    torch, capi = _mods()
    e = lambda *s, **k: torch.empty(s, device="cuda", **k)  # noqa: E731
    q, s = capi.quantize_blocks(ctx, e(0, 300).half())
    assert q.shape == (0, 300) and s.shape == (3, 0)
    w, sw = capi.quantize_blocks(ctx, torch.randn((5, 300), device="cuda"), 128)
    assert capi.fp8_matmul(ctx, q, s, w, sw).shape == (0, 5)
    r, n = capi.residual_norm(ctx, e(0, 64), e(0, 64), weight=torch.ones(64, device="cuda"))
    assert r.shape == n.shape == (0, 64)
    lp, ent, tl, tt = capi.token_logprobs(ctx, e(0, 10), e(0, 2, dtype=torch.int32), top=3)
    assert lp.shape == (0, 2) and ent.shape == (0,) and tt.shape == (0, 3)
    ctx.sync_check()


def test_refusals(ctx):
    torch, capi = _mods()
    x = torch.randn((8, 256), device="cuda")
    q, s = capi.quantize_blocks(ctx, x)
    w, sw = capi.quantize_blocks(ctx, x, 128)
    ones = torch.ones(256, device="cuda")
    tokens = torch.zeros((8, 1), device="cuda", dtype=torch.int32)
    bad = [
        lambda: capi.quantize_blocks(ctx, x.int()),
        lambda: capi.quantize_blocks(ctx, x, block_rows=64),
        lambda: capi.quantize_blocks(ctx, x.t()),
        lambda: capi.quantize_blocks(ctx, x.cpu()),
        lambda: capi.quantize_blocks(ctx, x, q=q[:4]),
        lambda: capi.quantize_blocks(ctx, x[:, :100], q=torch.empty((8, 100), device="cuda", dtype=torch.float8_e4m3fn)),
        lambda: capi.quantize_blocks(ctx, x, scales=s[:, :4]),
        lambda: capi.fp8_matmul(ctx, q, s, w[:, :128], sw),
        lambda: capi.fp8_matmul(ctx, q, s[:, :7], w, sw),
        lambda: capi.fp8_matmul(ctx, q, s, w, s),
        lambda: capi.fp8_matmul(ctx, q, s, w, sw, bias=ones),
        lambda: capi.fp8_matmul(ctx, q, s, w, sw, out_dtype=capi.EXB_I32),
        lambda: capi.fp8_matmul(ctx, x, s, w, sw),
        lambda: capi.fp8_matmul(ctx, torch.empty(8 * 256 + 16, device="cuda", dtype=torch.uint8)[1:1 + 8 * 256].view(torch.float8_e4m3fn).view(8, 256), s, w, sw),
        lambda: capi.residual_norm(ctx, x, x[:, :128].contiguous(), weight=ones),
        lambda: capi.residual_norm(ctx, x, x.half(), weight=ones),
        lambda: capi.residual_norm(ctx, x, x, weight=ones[:128]),
        lambda: capi.residual_norm(ctx, x, x, weight=ones, eps=-1.0),
        lambda: capi.residual_norm(ctx, x, x, weight=ones, kind=2),
        lambda: capi.residual_norm(ctx, x, x, weight=ones, gate=x[:2], gate_rows=3),
        lambda: capi.residual_norm(ctx, x, x, weight=ones, post_bias=ones),
        lambda: capi.residual_norm(ctx, x, x, weight=ones, r=x, n=x),
        lambda: capi.residual_norm(ctx, torch.zeros((1, 40000), device="cuda"), weight=torch.ones(40000, device="cuda")),
        lambda: capi.token_logprobs(ctx, x, tokens, top=33),
        lambda: capi.token_logprobs(ctx, x[:, :4], tokens, top=5),
        lambda: capi.token_logprobs(ctx, x, tokens, top=-1),
        lambda: capi.token_logprobs(ctx, x, tokens.long()),
        lambda: capi.token_logprobs(ctx, x, tokens[:4]),
        lambda: capi.token_logprobs(ctx, x, tokens, scale=0.0),
        lambda: capi.token_logprobs(ctx, x, tokens, scale=math.nan),
        lambda: capi.token_logprobs(ctx, x.int(), tokens),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(capi.ExbError) as e:
            call()
        assert e.value.code in (capi.EXB_ERR_BAD_ARG, capi.EXB_ERR_UNSUPPORTED), i
    ctx.sync_check()
    # null buffers and descriptors, at the C entries
    import ctypes as C
    L, h, E = capi.lib(), ctx.handle, capi.EXB_ERR_BAD_ARG
    xp, qp, sp, wp, swp = (v.data_ptr() for v in (x, q, s, w, sw))

    def blocks(**k):
        return C.byref(capi.BlocksDesc(**{**dict(rows=8, C=256, in_dtype=capi.EXB_F32, block_rows=1, x_stride=256, q_stride=256, scale_stride=8), **k}))
    assert L.exb_quantize_blocks_fwd(h, blocks(), None, qp, sp, None) == E
    assert L.exb_quantize_blocks_fwd(None, blocks(), xp, qp, sp, None) == E
    assert L.exb_quantize_blocks_fwd(h, None, xp, qp, sp, None) == E
    for k in (dict(x_stride=255), dict(q_stride=200), dict(q_stride=264), dict(scale_stride=7), dict(rows=-1), dict(C=0), dict(in_dtype=capi.EXB_I8)):
        assert L.exb_quantize_blocks_fwd(h, blocks(**k), xp, qp, sp, None) == E, k

    def matmul(**k):
        return C.byref(capi.MatmulDesc(**{**dict(M=8, N=8, K=256, y_dtype=capi.EXB_F16, a_stride=256, a_scale_stride=8, w_stride=256, w_scale_stride=2, y_stride=8), **k}))
    assert L.exb_fp8_matmul_fwd(h, matmul(), qp, sp, wp, swp, None, None, None) == E
    assert L.exb_fp8_matmul_fwd(h, None, qp, sp, wp, swp, None, xp, None) == E
    for k in (dict(K=0), dict(N=0), dict(M=-1), dict(a_stride=240), dict(w_stride=250), dict(y_stride=7), dict(w_scale_stride=1), dict(y_dtype=capi.EXB_I8)):
        assert L.exb_fp8_matmul_fwd(h, matmul(**k), qp, sp, wp, swp, None, xp, None) == E, k
    assert L.exb_residual_norm_fwd(h, None, xp, *[None] * 10) == E

    def scores(**k):
        return C.byref(capi.LogprobsDesc(**{**dict(rows=8, stride=256, V=256, dtype=capi.EXB_F32, n_given=0, top=0, scale=1.0), **k}))
    assert L.exb_token_logprobs_fwd(h, scores(), None, None, None, sp, None, None, None) == E
    assert L.exb_token_logprobs_fwd(h, None, xp, None, None, sp, None, None, None) == E
    for k in (dict(n_given=1), dict(top=1), dict(stride=255), dict(V=0), dict(rows=-1), dict(scale=-1.0), dict(top=-1), dict(dtype=capi.EXB_I32)):
        assert L.exb_token_logprobs_fwd(h, scores(**k), xp, None, None, sp, None, None, None) == E, k
    ctx.sync_check()


# ---- together ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,C,V", [(1, 512, 4001), (70, 1000, 1000), (300, 256, 9000)])
def test_token_head(ctx, rows, C, V):
    """Norm, e4m3, product and log probabilities one after the other: each against 64 bits on what the one before it wrote."""
    torch, capi = _mods()
    from excalibur_b200.token_head import TokenHead
    g = _gen(rows)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    w = 1 + 0.1 * rand(C)
    head = TokenHead(ctx, rand(V, C).half() * 0.1, w, residual_scale=0.5)
    h, x = rand(rows, C).half(), rand(rows, C).half()
    tokens = torch.randint(0, V, (rows, 2), device="cuda", generator=g).int()
    r, logits = head.logits(h, x, out_dtype=capi.EXB_F32)
    r2, q, s = capi.residual_norm(ctx, h, x, residual_scale=0.5, weight=w, quantized=True)
    ctx.sync_check()
    assert torch.equal(r, r2)
    _check_product(logits, q, s, head.weights, head.scales, None, "float32")
    given, entropy, best, best_tokens = head.scores(h, x, tokens, top=5, temperature=2.0, out_dtype=capi.EXB_F32)
    again = capi.token_logprobs(ctx, logits, tokens, top=5, scale=0.5)
    ctx.sync_check()
    assert all(torch.equal(a, b) for a, b in zip((given, entropy, best, best_tokens), again))
    _check_logprobs(ctx, logits, tokens, 5, 0.5)
    # and the whole against the same without 8 bits: e4m3 is off by 2^-4 of each factor at most, which random signs average out
    ref = (x.double() + 0.5 * h.double())
    ref = ref * (ref.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w.double()
    full = ref @ (_dequantized(head.weights, head.scales, 128)).t()
    assert ((logits.double() - full).norm() / full.norm()) < 0.04


def test_token_head_example_runs(ctx, capsys, monkeypatch):
    from excalibur_b200 import token_head
    monkeypatch.setattr("sys.argv", ["token_head", "--rows", "3", "--channels", "256", "--vocab", "1000", "--top", "2"])
    token_head.main()
    lines = capsys.readouterr().out.strip().split("\n")
    assert len(lines) == 3 and all(" best " in line for line in lines)
