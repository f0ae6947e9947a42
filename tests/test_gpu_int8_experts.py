"""8-bit integers by row, their product, and products grouped by expert, against plain implementations in 64 bits, at the sizes, strides, types and
groups where they can go wrong."""
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


def _rows(t, pad=0, offset=0, fill=7):
    """The same matrix in rows that are pad elements further apart and start offset elements into their buffer."""
    import torch
    if not pad and not offset:
        return t
    buf = torch.full((t.shape[0] * (t.shape[1] + pad) + offset,), fill, device=t.device, dtype=t.dtype)
    v = buf[offset:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


# ---- rows in 8-bit integers ----------------------------------------------------------------------------------------------

def _ref_rows(x):
    """The definition: scales and their reciprocals in IEEE fp32, products exact in 64 bits."""
    import torch
    x = x.float().cpu()
    largest = x.abs().amax(1)
    scale = torch.maximum(largest / torch.tensor(127.0), torch.tensor(2.0 ** -126))
    q = torch.round(x.double() * (torch.tensor(1.0) / scale).double()[:, None])
    bad = ~torch.isfinite(x).all(1)
    scale[bad] = math.nan
    q[bad] = 0
    return q.to(torch.int8), scale


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 255), (9, 256), (8, 257), (17, 512), (33, 513), (2, 1000), (64, 2048), (7, 2049), (1, 4096), (12, 4097), (300, 768),
          (3, 8192), (2, 8200), (4, 16384), (5, 16385), (1, 40000), (2, 70001)]


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows(ctx, rows, C, dtype):
    torch, capi = _mods()
    x = torch.randn((rows, C), device="cuda", generator=_gen(rows * 7 + C)) * 3
    x[:, C // 2] *= 50
    x[0] *= 1e-3
    x = x.to(getattr(torch, dtype))
    rq, rs = _ref_rows(x)
    for pad, offset in ((0, 0), (3, 1), (16, 8), (1, 0)):
        q, s = capi.quantize_rows(ctx, _rows(x, pad, offset))
        ctx.sync_check()
        assert torch.equal(s.cpu(), rs)
        assert torch.equal(q.cpu(), rq)
    # against 64 bits: half a step, and what scale and reciprocal are rounded by (2^-24 of up to 127 steps each)
    assert ((q.double() * s.double()[:, None] - x.double()).abs() <= s.double()[:, None] * (0.5 + 127 * 2.0 ** -22)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [64, 300, 3001, 20000])
def test_quantize_rows_at_the_ends_of_the_types(ctx, dtype, C):
    torch, capi = _mods()
    t = getattr(torch, dtype)
    x = torch.zeros((12, C), device="cuda", dtype=t)
    x[1] = torch.finfo(t).max
    x[2] = -torch.finfo(t).max
    x[3, C - 1] = torch.finfo(t).tiny
    x[4, 0] = torch.finfo(t).smallest_normal * torch.finfo(t).eps      # the smallest number there is
    x[5, C // 2], x[5, 0] = math.inf, 3
    x[6, C - 1], x[6, 0] = -math.inf, 3
    x[7, C // 3], x[7, 0] = math.nan, 3
    x[8] = -0.0
    x[9] = torch.arange(C, device="cuda").to(t) % 255 / 2 - 63.5      # ties, where the scale is a half
    x[9, 0] = 63.5
    x[10, C - 1] = -1
    for pad in (0, 1):
        q, s = capi.quantize_rows(ctx, _rows(x, pad, pad))
        ctx.sync_check()
        rq, rs = _ref_rows(x)
        assert torch.equal(torch.isnan(s.cpu()), torch.isnan(rs)) and torch.equal(torch.nan_to_num(s.cpu()), torch.nan_to_num(rs))
        assert torch.equal(q.cpu(), rq)


def test_quantize_rows_leaves_what_lies_between_rows(ctx):
    torch, capi = _mods()
    for C in (1, 100, 127, 250, 2050):
        x = torch.randn((37, C), device="cuda", generator=_gen(C)).half()
        wide = torch.full((38, 2064), 0x55, device="cuda", dtype=torch.int8)
        scales = torch.full((40,), -1.0, device="cuda")
        capi.quantize_rows(ctx, x, q=wide[:37, :C], scales=scales[:37])
        ctx.sync_check()
        assert (wide[:, C:] == 0x55).all() and (wide[37] == 0x55).all()
        assert (scales[:37] > 0).all() and (scales[37:] == -1).all()


# ---- products ------------------------------------------------------------------------------------------------------------

def _int8(shape, seed):
    """Whole numbers in rows that start at multiples of 16 bytes; what lies behind a row's end would show."""
    import torch
    pitch = (shape[-1] + 15) // 16 * 16
    wide = torch.full((*shape[:-1], pitch), 99, device="cuda", dtype=torch.int8)
    wide[..., :shape[-1]] = torch.randint(-128, 128, shape, device="cuda", generator=_gen(seed), dtype=torch.int32).to(torch.int8)
    return wide[..., :shape[-1]]


def _check_int8(y, a, sa, w, sw, bias, dtype):
    """Sum and product of scales are rounded to fp32, then the product with the bias' sum: 2^-24 each of what is added in magnitude, and the result's type."""
    import torch
    product = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()
    ref = product if bias is None else product + bias.double()
    mag = product.abs() + (0 if bias is None else bias.double().abs())
    tol = (4 * 2.0 ** -24 * mag + ROUND[dtype] * ref.abs()) * (1 + 2.0 ** -10) + (SMALLEST_HALF if dtype == "float16" else 2.0 ** -149)
    assert y.shape == ref.shape and torch.isfinite(y).all()
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


SIZES = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (1, 1000, 1234), (2, 257, 129), (5, 64, 16), (7, 130, 4096), (16, 512, 640), (17, 1000, 384), (31, 384, 2000),
         (33, 129, 300), (48, 2048, 1024), (64, 4096, 512), (65, 300, 1000), (100, 1408, 768), (128, 128, 128), (129, 129, 129), (200, 1000, 1111),
         (256, 256, 256), (257, 511, 400), (333, 1000, 1234), (512, 1024, 2048), (700, 2500, 200), (1000, 777, 999), (2048, 2048, 1024), (1500, 4000, 500),
         (4100, 300, 260), (300, 9000, 140), (40, 40000, 300), (3, 30000, 1290), (9, 130, 1750), (15, 4900, 1540), (50, 9001, 777), (100, 2500, 1700)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_int8_matmul(ctx, M, N, K, dtype):
    torch, capi = _mods()
    g = _gen(M * 31 + N * 7 + K)
    a, w = _int8((M, K), M + N), _int8((N, K), M + K)
    sa = torch.rand(M, device="cuda", generator=g) * 0.01 + 1e-4
    sw = torch.rand(N, device="cuda", generator=g) * 0.01 + 1e-4
    bias = torch.randn(N, device="cuda", generator=g) if (M + N) % 2 else None
    dt = capi.exb_dtype_of(getattr(torch, dtype))
    y = capi.int8_matmul(ctx, a, sa, w, sw, bias, dt)
    again = capi.int8_matmul(ctx, a, sa, w, sw, bias, dt)
    ctx.sync_check()
    _check_int8(y, a, sa, w, sw, bias, dtype)
    assert torch.equal(y, again)


@pytest.mark.parametrize("M", [1, 40, 100, 600])
def test_int8_matmul_of_the_longest_sums(ctx, M):
    """The largest sum that an int32 holds, and its neighbours of either sign."""
    torch, capi = _mods()
    K, N = 131071, 130
    a = torch.full((M, K + 1), -128, device="cuda", dtype=torch.int8)[:, :K]
    w = torch.full((N, K + 1), -128, device="cuda", dtype=torch.int8)[:, :K]
    w[1::2] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = capi.int8_matmul(ctx, a, one[:M], w, one[:N], None, capi.EXB_F32)
    ctx.sync_check()
    _check_int8(y, a, one[:M], w, one[:N], None, "float32")
    assert (y[:, 0] > 0).all() and (y[:, 1] < 0).all()


@pytest.mark.parametrize("M,N,K", [(3, 200, 300), (70, 200, 300), (300, 700, 1000), (600, 1100, 300)])
def test_int8_matmul_takes_strides_and_writes_nothing_else(ctx, M, N, K):
    torch, capi = _mods()
    g = _gen(5)
    a = _rows(_int8((M, K), 1).contiguous(), (-K) % 16 + 32, 0, 99)
    w = _rows(_int8((N, K), 2).contiguous(), (-K) % 16 + 16, 0, 99)
    sa, sw = torch.rand(M, device="cuda", generator=g), torch.rand(N, device="cuda", generator=g)
    for dtype in DTYPES:
        for offset, pad in ((0, 8), (1, 3), (0, 0)):
            if dtype == "float16":      # (sums of up to 127^2 * 1000 are beyond its range)
                s = sa * 1e-5
            else:
                s = sa
            buf = torch.full((M * (N + pad) + offset,), 77, device="cuda", dtype=getattr(torch, dtype))
            wide = buf[offset:].view(M, N + pad)
            y = capi.int8_matmul(ctx, a, s, w, sw, None, capi.exb_dtype_of(buf), y=wide[:, :N])
            ctx.sync_check()
            _check_int8(y, a, s, w, sw, None, dtype)
            assert (wide[:, N:] == 77).all() and (buf[:offset] == 77).all()


@pytest.mark.parametrize("M", [1, 40, 200, 600])
def test_int8_matmul_of_rows_without_a_scale(ctx, M):
    """A row that held a NaN or an infinity is NaN in all its results, and in no other row's."""
    torch, capi = _mods()
    x = torch.randn((M, 300), device="cuda", generator=_gen(M))
    x[M // 2, 7] = math.inf
    a, sa = capi.quantize_rows(ctx, x)
    w, sw = capi.quantize_rows(ctx, torch.randn((200, 300), device="cuda", generator=_gen(M + 1)))
    y = capi.int8_matmul(ctx, a, sa, w, sw, None, capi.EXB_F32)
    ctx.sync_check()
    assert torch.isnan(y[M // 2]).all()
    keep = [i for i in range(M) if i != M // 2]
    if keep:
        _check_int8(y[keep], a[keep], sa[keep], w, sw, None, "float32")


# ---- products grouped by expert --------------------------------------------------------------------------------------------

def _check_float(y, a, w, bias, dtype):
    """K products and their sums in fp32: each is off by a unit in the last place (2^-23) at most of what has been added in magnitude; then the result's type."""
    import torch
    A, W = a.double(), w.double()
    ref, mag = A @ W.t(), A.abs() @ W.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    tol = (a.shape[1] + 8) * 2.0 ** -23 * mag + ROUND[dtype] * ref.abs() + (SMALLEST_HALF if dtype == "float16" else 0)
    assert torch.isfinite(y).all()
    err = (y.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


def _counts(kind, M, E):
    import random
    r = random.Random(M * 1000 + E)
    if kind == "one":                   # all rows are one expert's
        c = [0] * E
        c[r.randrange(E)] = M
    elif kind == "even":
        c = [M // E + (i < M % E) for i in range(E)]
    else:                               # some without a row, one with many
        c = [0] * E
        for _ in range(M):
            c[min(int(abs(r.gauss(0, E / 4))), E - 1)] += 1
        r.shuffle(c)
    return c


def _grouped_case(ctx, M, N, K, E, kind, types, tail=0, bias=True):
    torch, capi = _mods()
    dtype, out = types
    g = _gen(M + N + K + E)
    counts = _counts(kind, M, E)
    ends = torch.tensor(counts).cumsum(0).int().cuda()
    if dtype == "int8":
        a, w = _int8((M + tail, K), 3), _int8((E, N, K), 4)
        sa, sw = torch.rand(M + tail, device="cuda", generator=g) * 1e-3, torch.rand((E, N), device="cuda", generator=g) * 1e-2
    else:
        t = getattr(torch, dtype)
        a = torch.randn((M + tail, K), device="cuda", generator=g).to(t)
        w = (torch.randn((E, N, K), device="cuda", generator=g) * 0.1).to(t)
        sa = sw = None
    b = torch.randn((E, N), device="cuda", generator=g) if bias else None
    y = torch.full((M + tail, N), 77.0, device="cuda", dtype=getattr(torch, out))
    capi.grouped_matmul(ctx, a, w, ends, sa, sw, b, capi.exb_dtype_of(y), y=y)
    again = capi.grouped_matmul(ctx, a, w, ends, sa, sw, b, capi.exb_dtype_of(y))
    ctx.sync_check()
    assert torch.equal(again[:M], y[:M])
    assert (y[M:] == 77).all()
    first = 0
    for e, n in enumerate(counts):
        if n:
            s = slice(first, first + n)
            be = None if b is None else b[e]
            if dtype == "int8":
                _check_int8(y[s], a[s], sa[s], w[e], sw[e], be, out)
            else:
                _check_float(y[s], a[s], w[e], be, out)
        first += n


TYPES = [("int8", "float16"), ("int8", "float32"), ("int8", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("bfloat16", "float32")]


@pytest.mark.parametrize("M,N,K,E", [
    (1, 1, 8, 1), (1, 300, 128, 4), (2, 512, 512, 8), (7, 130, 200, 3), (40, 256, 136, 64), (100, 300, 264, 16), (129, 200, 1000, 5), (257, 513, 64, 2),
    (509, 1500, 400, 64), (300, 136, 1032, 33), (1000, 250, 328, 7), (2000, 700, 256, 8), (3000, 1100, 136, 40), (512, 512, 512, 1), (777, 128, 8, 200)])
@pytest.mark.parametrize("kind", ["one", "even", "uneven"])
@pytest.mark.parametrize("types", TYPES)
def test_grouped_matmul(ctx, M, N, K, E, kind, types):
    _grouped_case(ctx, M, N, K, E, kind, types, tail=3 if M % 2 else 0, bias=N % 2 == 0)


@pytest.mark.parametrize("M,N,K,E", [(5, 300, 77, 3), (200, 129, 129, 9), (900, 1001, 333, 4)])
def test_grouped_matmul_of_odd_widths_in_int8(ctx, M, N, K, E):
    for kind in ("even", "uneven"):
        _grouped_case(ctx, M, N, K, E, kind, ("int8", "float16"), tail=1)


@pytest.mark.parametrize("types", TYPES)
def test_grouped_matmul_of_many_experts(ctx, types):
    _grouped_case(ctx, 1500, 40, 64, 1024, "uneven", types, tail=5)
    _grouped_case(ctx, 3, 40, 64, 1024, "uneven", types)


@pytest.mark.parametrize("M", [4, 300, 2000])
def test_grouped_matmul_of_ends_that_are_not_in_order(ctx, M):
    """One below those before it counts as theirs, one above the rows as their number; without any rows nothing is written."""
    torch, capi = _mods()
    g = _gen(M)
    a = torch.randn((M, 64), device="cuda", generator=g).half()
    w = torch.randn((4, 96, 64), device="cuda", generator=g).half()
    h = M // 2
    for ends, meant in (([h, h - 1, M + 5, M], [h, h, M, M]), ([-3, 0, h, 2 ** 31 - 1], [0, 0, h, M]), ([M, 0, 0, 0], [M] * 4), ([0, 0, 0, 0], [0] * 4),
                        ([-2 ** 31, -1, -1, -5], [0] * 4)):
        y = torch.full((M, 96), 77.0, device="cuda", dtype=torch.float16)
        capi.grouped_matmul(ctx, a, w, torch.tensor(ends, dtype=torch.int32, device="cuda"), y=y)
        ctx.sync_check()
        first = 0
        for e, end in enumerate(meant):
            if end > first:
                _check_float(y[first:end], a[first:end], w[e], None, "float16")
            first = end
        assert (y[meant[-1]:] == 77).all()


def test_grouped_matmul_takes_strides(ctx):
    """Rows and experts that are apart, a result inside a wider one, rows that start anywhere."""
    torch, capi = _mods()
    for M in (30, 400, 1500):
        for dtype in ("float16", "bfloat16"):
            t = getattr(torch, dtype)
            g = _gen(M)
            room = torch.full((3, 70, 160), math.nan, device="cuda", dtype=t)
            w = room[:, :61, :120]
            w.copy_(torch.randn((3, 61, 120), device="cuda", generator=g))
            a = _rows(torch.randn((M, 120), device="cuda", generator=g).to(t), 24, 8, math.nan)
            ends = torch.tensor([M // 3, M // 3, M - 1], dtype=torch.int32, device="cuda")
            wide = torch.full((M, 80), 77.0, device="cuda", dtype=t)
            for offset in (0, 1, 8):
                wide.fill_(77)
                y = wide[:, offset:offset + 61]
                capi.grouped_matmul(ctx, a, w, ends, y=y)
                ctx.sync_check()
                _check_float(y[:M // 3], a[:M // 3], w[0], None, dtype)
                _check_float(y[M // 3:M - 1], a[M // 3:M - 1], w[2], None, dtype)
                assert (y[M - 1] == 77).all() and (wide[:, :offset] == 77).all() and (wide[:, offset + 61:] == 77).all()


def test_grouped_matmul_keeps_what_is_not_a_number_in_its_row(ctx):
    torch, capi = _mods()
    for M in (20, 300, 1200):
        a = torch.randn((M, 128), device="cuda", generator=_gen(M)).half()
        a[M // 2, 5] = math.nan
        a[M // 4, 100] = math.inf
        w = torch.rand((2, 200, 128), device="cuda", generator=_gen(1)).half() + 0.5
        ends = torch.tensor([M // 2 + 3, M], dtype=torch.int32, device="cuda")
        y = capi.grouped_matmul(ctx, a, w, ends, out_dtype=capi.EXB_F32)
        ctx.sync_check()
        assert torch.isnan(y[M // 2]).all() and (y[M // 4] == math.inf).all()
        fine = torch.isfinite(y).all(1)
        assert int((~fine).sum()) == 2
    w[0, 3, 7] = math.nan      # an expert's weights: in its rows' one channel only
    y = capi.grouped_matmul(ctx, torch.ones_like(a), w, ends, out_dtype=capi.EXB_F32)
    ctx.sync_check()
    bad = torch.isnan(y)
    assert bad[:M // 2 + 3, 3].all() and int(bad.sum()) == M // 2 + 3


# ---- together, on streams and in graphs ------------------------------------------------------------------------------------

def _block(capi, ctx, x, up, down, ends):
    """A feed-forward block by experts in 8-bit integers, as a program runs it."""
    import torch
    q, s = capi.quantize_rows(ctx, x)
    h = capi.grouped_matmul(ctx, q, up[0], ends, s, up[1])
    h = torch.relu(h)
    q, s = capi.quantize_rows(ctx, h)
    return capi.grouped_matmul(ctx, q, down[0], ends, s, down[1])


def _weights(capi, ctx, E, N, K, seed):
    import torch
    w = torch.randn((E * N, K), device="cuda", generator=_gen(seed)) * K ** -0.5
    q, s = capi.quantize_rows(ctx, w)
    return q.unflatten(0, (E, N)), s.view(E, N)


@pytest.mark.parametrize("M", [6, 200])
def test_a_block_by_experts(ctx, M):
    """Against the same block without rounding: each of two quantisations is off by half a step of its row's largest, 1 in 254, so that a result is off by a
    few per cent of the results' spread."""
    torch, capi = _mods()
    E, C, H = 4, 256, 512
    up, down = _weights(capi, ctx, E, H, C, 1), _weights(capi, ctx, E, C, H, 2)
    x = torch.randn((M, C), device="cuda", generator=_gen(3)).half()
    ends = torch.tensor([M // 2, M // 2, M - 1, M], dtype=torch.int32, device="cuda")
    y = _block(capi, ctx, x, up, down, ends)
    ctx.sync_check()
    first = 0
    for e, end in enumerate(ends.tolist()):
        W1, W2 = up[0][e].double() * up[1][e].double()[:, None], down[0][e].double() * down[1][e].double()[:, None]
        ref = torch.relu(x[first:end].double() @ W1.t()) @ W2.t()
        if end > first:
            assert ((y[first:end].double() - ref).norm() / ref.norm()) < 0.05
        first = end


def test_streams_and_graphs(ctx):
    """Another stream, a captured chain that is replayed with new inputs, and two graphs in turn."""
    torch, capi = _mods()
    E, C, H, M = 3, 192, 320, 37
    up, down = _weights(capi, ctx, E, H, C, 1), _weights(capi, ctx, E, C, H, 2)
    ends = torch.tensor([10, 30, 37], dtype=torch.int32, device="cuda")
    xs = [torch.randn((M, C), device="cuda", generator=_gen(i)).half() for i in range(3)]
    want = [_block(capi, ctx, x, up, down, ends) for x in xs]
    w, sw = _weights(capi, ctx, 1, 500, C, 5)
    dense = [capi.int8_matmul(ctx, *capi.quantize_rows(ctx, x), w[0], sw[0]) for x in xs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _block(capi, ctx, xs[1], up, down, ends)
        got_dense = capi.int8_matmul(ctx, *capi.quantize_rows(ctx, xs[1]), w[0], sw[0])
        ctx.sync_check()
    assert torch.equal(got, want[1]) and torch.equal(got_dense, dense[1])
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _block(capi, ctx, x, up, down, ends)
            z = capi.int8_matmul(ctx, *capi.quantize_rows(ctx, x), w[0], sw[0])
        graphs.append((g, x, y, z))
    for turn in range(4):
        for i, (g, x, y, z) in enumerate(graphs):
            x.copy_(xs[(turn + i) % 3])
            g.replay()
        torch.cuda.synchronize()
        for i, (g, x, y, z) in enumerate(graphs):
            assert torch.equal(y, want[(turn + i) % 3]) and torch.equal(z, dense[(turn + i) % 3])
    ctx.sync_check()


def test_kernels_follow_each_other_without_a_wait(ctx):
    """Many dependent calls in a row: each starts while the one before it ends, and reads what that has written."""
    torch, capi = _mods()
    C = 512
    w, sw = _weights(capi, ctx, 1, C, C, 9)
    for M in (1, 50, 300):
        x = torch.randn((M, C), device="cuda", generator=_gen(M)).half()
        outs = []
        for synchronous in (False, True):
            h = x
            for _ in range(20):
                q, s = capi.quantize_rows(ctx, h)
                if synchronous:
                    torch.cuda.synchronize()
                h = capi.int8_matmul(ctx, q, s, w[0], sw[0])
                if synchronous:
                    torch.cuda.synchronize()
            outs.append(h)
        ctx.sync_check()
        assert torch.isfinite(outs[0]).all() and torch.equal(*outs)


def test_another_device_than_the_current_one_is_refused(ctx):
    torch, capi = _mods()
    x = torch.randn((4, 64)).half()      # on the host
    with pytest.raises(capi.ExbError):
        capi.quantize_rows(ctx, x)
    q, s = capi.quantize_rows(ctx, x.cuda())
    with pytest.raises(capi.ExbError):
        capi.int8_matmul(ctx, q, s, q.cpu(), s)
    with pytest.raises(capi.ExbError):
        capi.int8_matmul(ctx, q, s.cpu(), q, s)
    with pytest.raises(capi.ExbError):
        capi.grouped_matmul(ctx, x.cuda(), x.cuda()[None], torch.tensor([4], dtype=torch.int32))
    ctx.sync_check()
