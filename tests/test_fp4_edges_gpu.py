"""4-bit kernels where several of their mechanisms meet: K split inside clusters, rings that wrap, lists that say more than
they hold, factors at the ends of their range."""

import ctypes

import pytest
import torch

from arcticinference_b200 import build, ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

import fp4_calls
from fp4_util import FORMATS, oracle_rows, oracle_values, routing_of
from test_fp4_gpu import _check

pytestmark = pytest.mark.gpu


def _rand(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


def test_clusters_of_two_streams():
    """Products whose K is split, on two streams at once: CTAs of both share SMs."""
    w = [quant.quantize_weight_fp4(_rand(4096, 4096, seed=i, scale=0.02).cuda(), f) for i, f in enumerate(FORMATS)]
    x = [_rand(m, 4096, seed=5 + i).cuda() for i, m in enumerate((1, 100))]
    want = [ops.linear(a, b) for a, b in zip(x, w)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear(x[i], w[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])
    ops.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_tiles_counted_than_listed(fmt):
    """A count beyond the list: nothing behind the list, or behind the scales that belong to it, is touched."""
    counts = [100, 0, 60, 129]
    n, K = sum(counts), 160
    x = _rand(n, K, seed=1).cuda()
    w4 = quant.quantize_weight_fp4(_rand(4, 64, K, seed=2, scale=0.1).cuda(), fmt)
    for even in (False, True):
        r = routing_of(counts, "cuda", even, slack=0)
        want = stream_ops.grouped_linear(x, w4, r)
        for more in (1, 5, 100000):
            s = routing_of(counts, "cuda", even, slack=0)
            s.num_tiles += more
            q = ops.quant_fp4(x, fmt, s)
            assert torch.equal(q.dequantize(), ops.quant_fp4(x, fmt).dequantize())
            assert torch.equal(stream_ops.grouped_linear(q, w4, s), want)
            assert torch.equal(stream_ops.grouped_linear(x, w4, s), want)
        none = routing_of(counts, "cuda", even, slack=0)
        none.num_tiles.fill_(-3)
        out = torch.full((n, K), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.dequant_fp4(ops.quant_fp4(x, fmt, none), out=out)
        assert bool((out == 7).all())
    ops.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_routing_of_no_tokens(fmt):
    """Its list has no tiles: results without rows, as from the bf16 products."""
    E, N, K = 4, 64, 96
    w = _rand(E, N, K, seed=1, scale=0.1).cuda()
    w4 = quant.quantize_weight_fp4(w, fmt)
    i32 = dict(dtype=torch.int32, device="cuda")
    r = stream_ops.Routing(None, None, None, 1, E, torch.empty(0, 4, **i32), torch.zeros(1, **i32), counts=[0] * E)
    x = torch.empty(0, K, dtype=torch.bfloat16, device="cuda")
    for act, width in ((None, N), ("silu", N // 2)):
        got = stream_ops.grouped_linear(x, w4, r, act)
        assert got.shape == (0, width) == stream_ops.grouped_linear(x, w, r, act).shape
        q = ops.quant_fp4(x, fmt, r)
        assert stream_ops.grouped_linear(q, w4, r, act).shape == (0, width) and q.dequantize().shape == (0, K)
    with pytest.raises(ValueError):
        stream_ops.grouped_linear(torch.empty(0, K + 32, dtype=torch.bfloat16, device="cuda"), w4, r)
    ops.check_status()


def _relative_bound(x, w, y):
    """As product_bound, without the absolute term that it allows: half a bf16 step (2^-134 among the smallest numbers), fp32
    sums, the roundings of two factors."""
    mag = x.abs() @ w.abs().t()
    return (2.0 ** -8 + 2.0 ** -22) * y.abs() + (x.shape[1] / 16 + 8) * 2.0 ** -23 * mag + 2.0 ** -134


@pytest.mark.parametrize("M,K", [(1, 512), (20, 512), (5, 4096), (128, 4096), (150, 512), (300, 512)])
def test_factors_whose_product_leaves_the_range(M, K):
    """Factors of rows and features whose product fp32 does not hold, though that with the sum is an ordinary number."""
    fmt, N = "nvfp4", 264
    x, w = _rand(M, K, seed=1).abs(), _rand(N, K, seed=2).abs()
    x = (x.float() * 2.0 ** -100).to(torch.bfloat16)
    w = (w.float() * 2.0 ** -32).to(torch.bfloat16)
    w[1::3] = (w[1::3].float() * 2.0 ** 31).to(torch.bfloat16)           # beside ordinary features
    x[::2] = (x[::2].float() * 2.0 ** 99).to(torch.bfloat16)             # and ordinary rows
    w4 = quant.quantize_weight_fp4(w.cuda(), fmt)
    g, h = ops.quant_fp4(x.cuda(), fmt).row_scale, w4.row_scale
    assert M == 1 or float(g.min() * h.min()) == 0          # (2^-150 or less: half the smallest number)
    res, bias = torch.zeros(M, N, dtype=torch.bfloat16), torch.zeros(N, dtype=torch.bfloat16)
    xd, wd = oracle_rows(x, fmt).cuda(), oracle_values(w4.q, w4.scale, w4.row_scale, fmt).cuda()
    y = xd @ wd.t()
    assert float(y.min()) > 2.0 ** -126
    for kw in ({}, {"residual": res.cuda()}, {"bias": bias.cuda()}):
        got = ops.linear(x.cuda(), w4, **kw)
        bad = (got.double() - y).abs() > _relative_bound(xd, wd, y)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0], y[bad][0])
    ops.check_status()


@pytest.mark.parametrize("M,K", [(20, 512), (5, 4096), (150, 512), (300, 512)])
def test_sums_of_zero_beside_the_largest_factors(M, K):
    fmt, N = "nvfp4", 136
    x, w = torch.zeros(M, K, dtype=torch.bfloat16), torch.zeros(N, K, dtype=torch.bfloat16)
    x[:, 0], w[:, K - 1] = 2.0 ** 120, 2.0 ** 60
    x[:, 100], w[:, 100] = 1e-6, 1e-6          # (its code and scale are zero beside such numbers)
    w4 = quant.quantize_weight_fp4(w.cuda(), fmt)
    assert bool((ops.linear(x.cuda(), w4) == 0).all())
    assert bool((ops.linear(x.cuda(), w4, residual=torch.ones(M, N, dtype=torch.bfloat16, device="cuda")) == 1).all())
    ops.check_status()


@pytest.mark.parametrize("even", [False, True])
@pytest.mark.parametrize("act", [None, "silu"])
def test_experts_factors_whose_product_leaves_the_range(even, act):
    """Gate and up of ordinary size, reached through factors far from 1 on both sides."""
    fmt, N, K, counts = "nvfp4", 64, 256, [140, 0, 300, 7]
    n = sum(counts)
    x, w = _rand(n, K, seed=1).abs(), _rand(4, N, K, seed=2, scale=0.01).abs()
    small, large = (x.float() * 2.0 ** -110).to(torch.bfloat16), (w.float() * 2.0 ** 110).to(torch.bfloat16)
    tiny, little = (x.float() * 2.0 ** -100).to(torch.bfloat16), (w.float() * 2.0 ** -20).to(torch.bfloat16)
    for a, b in ((small, large), (tiny, little)):
        w4 = quant.quantize_weight_fp4(b.cuda(), fmt)
        got = stream_ops.grouped_linear(a.cuda(), w4, routing_of(counts, "cuda", even), act)
        first = 0
        for e, c in enumerate(counts):
            if c:
                xd = oracle_rows(a[first:first + c], fmt).cuda()
                wd = oracle_values(w4.q[e], w4.scale[e], w4.row_scale[e], fmt).cuda()
                y = xd @ wd.t()
                bound = _relative_bound(xd, wd, y)
                if act is not None:
                    g, u = (t.reshape(c, N // 2) for t in y.reshape(c, N // 32, 2, 16).unbind(2))
                    eg, eu = (t.reshape(c, N // 2) for t in
                              (bound - 2.0 ** -8 * y).reshape(c, N // 32, 2, 16).unbind(2))
                    y = g * torch.sigmoid(g) * u
                    # |d silu| < 1.1; exponential and division 2^-20 of the result; g, u >= 0
                    bound = 2.0 ** -8 * y + 1.1 * u * eg + g * eu + 2.0 ** -20 * y + 2.0 ** -134
                bad = (got[first:first + c].double() - y).abs() > bound
                assert not bad.any(), (e, int(bad.sum()), bad.nonzero()[0].tolist(), got[first:first + c][bad][0], y[bad][0])
            first += c
    ops.check_status()


@pytest.mark.parametrize("M,K", [(20, 512), (100, 4096), (300, 512)])
def test_rows_that_are_no_numbers_move_no_bit_of_others(M, K):
    N = 264
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), "nvfp4")
    g = (0.01 + torch.rand(N, generator=torch.Generator().manual_seed(3))).cuda()
    w4 = quant.Fp4Weight(w4.q, w4.scale, g, "nvfp4")
    x, bias = _rand(M, K, seed=2), _rand(N, seed=4, scale=10.0).cuda()
    clean = ops.linear(x.cuda(), w4, bias=bias)
    x[3, 7], x[M - 1, 200] = float("inf"), float("nan")
    got = ops.linear(x.cuda(), w4, bias=bias)
    assert got[[3, M - 1]].isnan().all()
    keep = [i for i in range(M) if i not in (3, M - 1)]
    assert torch.equal(got[keep], clean[keep])


def _all_refused(calls):
    for name, f in calls.items():
        with pytest.raises(ValueError):
            f()
            raise AssertionError("not refused: " + name)
    torch.cuda.synchronize()
    ops.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_refused_norms_and_activations(fmt):
    _all_refused(fp4_calls.norm_and_activation("cuda", fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_refused_products(fmt):
    _all_refused(fp4_calls.products("cuda", fmt))


# ------------------------------------------------------------------------ K split inside clusters, and rings that wrap
def _parts(M, N, K, fmt):
    P = ctypes.POINTER
    fn = build.load_kernels().ab200_linear_fp4_plan
    fn.argtypes = [ctypes.c_longlong] + [ctypes.c_int] * 4 + [P(ctypes.c_int), P(ctypes.c_int), P(ctypes.c_longlong)]
    parts, columns, smem = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert fn(M, N, K, FORMATS.index(fmt), sms, parts, columns, smem) == 0
    return parts.value


# (15 steps: parts of 8 and 7, or 4, 4, 4 and 3; 16, 18 and 56; 9 for few tokens: 5 and 4)
SPLIT = [(M, N, K) for M in (1, 7, 33, 64, 100, 128)
         for N, K in ((264, 3616), (264, 4096), (520, 4384), (520, 14336), (4096, 4096))] + [(1, 264, 2304), (33, 264, 2304)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", SPLIT)
def test_split_products(fmt, M, N, K):
    """The exchange of sums between the CTAs of a cluster, with everything that its epilogue does."""
    assert _parts(M, N, K, fmt) in (2, 4)
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=K ** -0.5).cuda(), fmt)
    wd = oracle_values(w4.q, w4.scale, w4.row_scale, fmt).cuda()
    x, bias, res = _rand(M, K, seed=2), _rand(N, seed=3), _rand(M, N, seed=4)
    _check(x, w4, fmt, wd=wd)
    _check(x, w4, fmt, bias=bias, wd=wd)
    _check(x, w4, fmt, bias=bias, act="gelu", wd=wd)
    _check(x, w4, fmt, residual=res, wd=wd)
    want = _check(x, w4, fmt, bias=bias, act="gelu", residual=res, wd=wd)
    place = res.cuda()
    got = ops.linear(x.cuda(), w4, bias=bias.cuda(), act="gelu", residual=place, out=place)
    assert got is place and torch.equal(got, want)
    buf = torch.full((M + 2, N + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.linear(x.cuda(), w4, bias=bias.cuda(), act="gelu", residual=res.cuda(), out=buf[1:M + 1, 8:N + 8])
    assert torch.equal(buf[1:M + 1, 8:N + 8], want)
    buf[1:M + 1, 8:N + 8] = 5.0
    assert bool((buf == 5).all())
    ops.check_status()


def test_split_products_have_both_numbers_of_parts():
    assert {_parts(M, N, K, fmt) for fmt in FORMATS for M, N, K in SPLIT} == {2, 4}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 70, 128])
def test_two_ctas_an_sm_whose_rings_wrap(fmt, M):
    """More tiles than SMs, and more steps than stages."""
    N, K = 19208, 4128
    assert _parts(M, N, K, fmt) == 1
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=K ** -0.5).cuda(), fmt)
    x, res = _rand(M, K, seed=2), _rand(M, N, seed=4)
    wd = oracle_values(w4.q, w4.scale, w4.row_scale, fmt).cuda()
    _check(x, w4, fmt, wd=wd)
    _check(x, w4, fmt, residual=res, bias=_rand(N, seed=3), wd=wd)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 520, 4096), (33, 4096, 4096), (128, 264, 2304), (100, 520, 512), (150, 520, 1056),
                                   (400, 520, 1056), (1000, 520, 1056)])
def test_a_row_gets_the_same_bits_wherever_it_stands(fmt, M, N, K):
    """Every run, and every order of a batch's rows."""
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), fmt)
    x = _rand(M, K, seed=2).cuda()
    first = ops.linear(x, w4)
    for i in range(4):
        order = torch.randperm(M, generator=torch.Generator().manual_seed(i)).cuda()
        assert torch.equal(ops.linear(x, w4), first)
        assert torch.equal(ops.linear(x[order], w4), first[order])


def test_every_scale_of_e4m3():
    """All 126 positive e4m3 numbers as block scales, each with values around every border of e2m1 in its units; and the
    largest values of a block around the borders between two scales."""
    scales = torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in scales.tolist():
        v = (borders[:, None] * torch.tensor([1 - 2.0 ** -7, 1.0, 1 + 2.0 ** -7])[None]).flatten() * s
        top = torch.full((1,), 6 * s)
        rows.append(torch.cat([top, v[:15], top, v[6:], torch.full((32,), 2688.0)]))
    both = (scales[:-1] + scales[1:]) / 2 * 6
    for b in both.tolist():
        for f in (1 - 2.0 ** -7, 1.0, 1 + 2.0 ** -7):
            rows.append(torch.cat([torch.full((32,), b * f), torch.full((32,), 2688.0)]))
    x = torch.stack(rows).to(torch.bfloat16)
    a = ops.quant_fp4(x.cuda(), "nvfp4")
    assert torch.equal(a.row_scale.cpu(), torch.ones(len(rows)))
    byte = quant.untile_fp4_scales(a.scale, len(rows), 4).cpu()
    assert set(byte[:126, 0].tolist()) == set(range(1, 127))
    assert torch.equal(oracle_values(a.q, a.scale, a.row_scale, "nvfp4"), oracle_rows(x, "nvfp4"))


@pytest.mark.parametrize("fmt", FORMATS)
def test_expansion_with_any_factors(fmt):
    """The same bits as on the CPU, also where a factor is no power of two and rounds on the way (8 million numbers: the
    other order of the two products changes 700000 of them in fp32)."""
    R, K = 2000, 4096
    gen = torch.Generator().manual_seed(2)
    q = torch.randint(0, 256, (R, K // 2), generator=gen, dtype=torch.uint8)
    low, high = (40, 72) if fmt == "nvfp4" else (120, 134)
    scale = torch.randint(low, high, quant.fp4_scale_tiles(R, K, fmt), generator=gen, dtype=torch.uint8)
    g = torch.rand(R, generator=gen) + 0.3
    g[::7] *= 2.0 ** -110
    g[1::7] *= 2.0 ** 100
    want = quant.Fp4Weight(q, scale, g, fmt).dequantize()
    got = quant.Fp4Weight(q.cuda(), scale.cuda(), g.cuda(), fmt).dequantize().cpu()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    v = oracle_values(q[:200], scale[:2], g[:200], fmt)          # bf16's rounding and two of fp32's
    assert ((got[:200].double() - v).abs() <= (2.0 ** -8 + 2.0 ** -22) * v.abs()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,inter,nblk", [(3, 40, 4), (1300, 8, 4), (130, 72, 12), (2, 24, 1364)])
def test_blocks_of_the_activation_that_end_inside_a_piece(fmt, M, inter, nblk):
    """A thread's 16 columns then belong to two (gate | up) blocks."""
    x = _rand(M, 2 * inter * nblk, seed=inter).cuda()
    a, b = ops.silu_mul_blocked(x, nblk, quant=fmt), ops.quant_fp4(ops.silu_mul_blocked(x, nblk), fmt)
    assert torch.equal(a.dequantize(), b.dequantize())
    want = oracle_rows(ops.silu_mul_blocked(x, nblk).cpu(), fmt)
    assert torch.equal(a.dequantize().cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_and_weights_that_are_parts_of_larger_ones(fmt):
    """Codes whose rows lie apart, of the rows and of the weight."""
    M, N, K = 70, 136, 256
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), fmt)
    q = ops.quant_fp4(_rand(M, K, seed=2).cuda(), fmt)
    want = ops.linear(q, w4)
    apart = lambda t: torch.cat([t, torch.full_like(t, 255)], 1)[:, :t.shape[1]]
    x2, w2 = quant.Fp4Rows(apart(q.q), q.scale, q.row_scale, fmt), quant.Fp4Weight(apart(w4.q), w4.scale, w4.row_scale, fmt)
    assert x2.q.stride(0) == K and w2.q.stride(0) == K
    assert torch.equal(ops.linear(x2, w2), want) and torch.equal(x2.dequantize(), q.dequantize())
    x3 = quant.Fp4Rows(apart(q.q[:1]), q.scale, None if q.row_scale is None else q.row_scale[:1], fmt)
    assert torch.equal(ops.linear(x3, w2), ops.linear(ops.quant_fp4(_rand(M, K, seed=2)[:1].cuda(), fmt), w4))


@pytest.mark.parametrize("fmt", FORMATS)
def test_residuals_that_overlap_the_output(fmt):
    _all_refused(fp4_calls.overlaps("cuda", fmt))
    for call, apart in fp4_calls.no_overlaps("cuda", fmt):
        want = apart()
        assert torch.equal(call(), want)
