"""The 4-bit kernels against the 64-bit oracle: quantisers bit for bit, products within the rounding of their result
and of fp32 sums."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

from fp4_util import FORMATS, oracle_rows, oracle_values, product_bound, routing_of, special_rows

pytestmark = pytest.mark.gpu


def _rand(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


def _codes(r):
    """Codes, one per byte; the sign of a zero says nothing."""
    q = r.q.cpu()
    c = torch.stack([q & 15, q >> 4], -1)
    return torch.where(c == 8, 0, c)


def _same(a, b):
    """Equal codes, scales of the rows that are there, and factors."""
    M = a.q.shape[0]
    blocks = a.shape[1] // quant.FP4_BLOCK[a.fmt]
    assert torch.equal(_codes(a), _codes(b))
    s, t = (quant.untile_fp4_scales(r.scale, M, -(-blocks // 4) * 4).cpu() for r in (a, b))
    assert torch.equal(s, t)          # (with the zeros that pad a row's last tile)
    if a.row_scale is not None:
        assert torch.equal(a.row_scale.cpu().view(torch.int32), b.row_scale.cpu().view(torch.int32))


# ------------------------------------------------------------------------ quantisers
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K", [(1, 32), (5, 96), (130, 4096), (1, 1024), (33, 1408), (3, 14336), (9, 8224), (2, 32768)])
def test_quantisation_is_bit_exact(fmt, M, K):
    x = _rand(M, K, seed=M + K)
    _same(ops.quant_fp4(x.cuda(), fmt), ops.quant_fp4(x, fmt))
    ops.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [32, 160, 2048])
def test_rows_at_the_formats_edges(fmt, K):
    x = special_rows(K, seed=K)
    a = ops.quant_fp4(x.cuda(), fmt)
    _same(a, ops.quant_fp4(x, fmt))
    want = oracle_rows(x, fmt)
    assert torch.equal(oracle_values(a.q, a.scale, a.row_scale, fmt), want)
    assert torch.equal(a.dequantize().cpu(), want.to(torch.bfloat16))


def test_every_pair_of_value_and_scale():
    """All bf16 mantissas against all e4m3 scales: blocks whose largest value fixes the scale, the others sweep the borders."""
    mant = torch.arange(128, 256).float()                                # 8-bit significands
    tops = (torch.arange(8, 16).float() / 8)[:, None] * 6 * 2.0 ** torch.arange(-4, 5).float()[None]
    rows = []
    for t in tops.flatten().tolist():
        v = (mant / 128)[:, None] * 2.0 ** torch.arange(-5, 3).float()[None] * t / 6
        v = v.flatten().clamp(max=t)[:1020].reshape(68, 15)
        rows.append(torch.cat([torch.full((v.shape[0], 1), t), v], 1).flatten())
    x = torch.stack(rows).to(torch.bfloat16)
    x = torch.cat([x, torch.full((x.shape[0], 32), 2688.0, dtype=torch.bfloat16)], 1)
    for fmt in FORMATS:
        a = ops.quant_fp4(x.cuda(), fmt)
        assert torch.equal(oracle_values(a.q, a.scale, a.row_scale, fmt), oracle_rows(x, fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_values_that_are_no_numbers(fmt):
    x = _rand(6, 4096)
    x[1, 5], x[2, 70], x[3, 4095] = float("nan"), float("inf"), float("-inf")
    a = ops.quant_fp4(x.cuda(), fmt)
    b = ops.quant_fp4(x, fmt)
    _same_nan = torch.equal(a.dequantize().cpu().isnan(), b.dequantize().isnan())
    assert _same_nan and torch.equal(_codes(a), _codes(b))
    fine = [0, 4, 5]
    assert torch.equal(a.dequantize().cpu()[fine], b.dequantize()[fine])


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_with_strides_and_odd_addresses(fmt):
    big = _rand(40, 4096 + 64).cuda()
    for x in (big[:, :4096], big[3:20, 64:], big[:, 1:97], big[::2, :128], big[:, :64].t().contiguous().t()):
        _same(ops.quant_fp4(x, fmt), ops.quant_fp4(x.cpu().contiguous(), fmt))
    r = ops.quant_fp4(big[:, :96], fmt)
    out = torch.empty(40, 96, dtype=torch.bfloat16, device="cuda")
    assert ops.dequant_fp4(r, out=out) is out and torch.equal(out.cpu(), ops.quant_fp4(big[:, :96].cpu(), fmt).dequantize())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K", [(1, 4096), (7, 64), (130, 2048), (3, 8224), (2, 16384)])
def test_norm_gives_the_rows_of_the_unfused_kernels(fmt, M, K):
    x, w, res = _rand(M, K).cuda(), (1 + 0.1 * _rand(K, seed=1)).cuda(), _rand(M, K, seed=2).cuda()
    r2 = res.clone()
    _same(ops.rmsnorm(x, w, 1e-5, quant=fmt), ops.quant_fp4(ops.rmsnorm(x, w, 1e-5), fmt))
    a = ops.rmsnorm(x, w, 1e-5, residual=res, quant=fmt)
    _same(a, ops.quant_fp4(ops.rmsnorm(x, w, 1e-5, residual=r2), fmt))
    assert torch.equal(res, r2)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,inter,nblk", [(1, 14336, 1), (9, 32, 1), (130, 1408, 1), (5, 48, 2), (3, 4096, 4), (2, 32768, 1)])
def test_activation_gives_the_rows_of_the_unfused_kernels(fmt, M, inter, nblk):
    x = _rand(M, 2 * inter * nblk, seed=inter).cuda()
    _same(ops.silu_mul_blocked(x, nblk, quant=fmt), ops.quant_fp4(ops.silu_mul_blocked(x, nblk), fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_sorted_by_expert(fmt):
    counts = [0, 5, 128, 0, 129, 1, 300, 0]
    n = sum(counts)
    for even in (False, True):
        r = routing_of(counts, "cuda", even)
        x = _rand(n + 9, 1408, seed=3)
        a = ops.quant_fp4(x.cuda(), fmt, r)
        out = torch.full((n + 9, 1408), 17.0, dtype=torch.bfloat16, device="cuda")
        ops.dequant_fp4(a, out=out)
        assert torch.equal(out.cpu()[:n], ops.quant_fp4(x[:n], fmt).dequantize())
        assert bool((out[n:] == 17).all())          # rows that no tile holds stay


# ------------------------------------------------------------------------ linear layers
def _check(x, w4, fmt, bias=None, residual=None, act=None, out=None, wd=None):
    got = ops.linear(x.cuda(), w4, bias=None if bias is None else bias.cuda(),
                     residual=None if residual is None else residual.cuda(), act=act, out=out)
    ops.check_status()
    xd = oracle_rows(x, fmt).cuda()
    wd = oracle_values(w4.q, w4.scale, w4.row_scale, fmt).cuda() if wd is None else wd
    y = xd @ wd.t()
    if bias is not None:
        y = y + bias.cuda().double()
    slack = torch.zeros((), dtype=torch.float64, device="cuda")
    if act == "gelu":
        y = torch.nn.functional.gelu(y)
        # the factors' products and GELU's own fp32 evaluation: a few steps of its argument, |gelu'| < 1.13
        slack = 0.13 * product_bound(xd, wd, torch.zeros_like(y)) + 2.0 ** -20 * (1 + y.abs())
    if residual is not None:
        y = y + residual.cuda().double()
    bound = product_bound(xd, wd, y) + slack
    if bias is not None:
        bound = bound + 2.0 ** -23 * bias.cuda().double().abs()
    bad = (got.double() - y).abs() > bound
    assert not bad.any(), "%d of %d off, first at %s: %g and %g" % (
        int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0], y[bad][0])
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [
    (1, 128, 256), (128, 128, 256), (1, 8, 32), (3, 120, 96), (16, 136, 160), (17, 392, 288), (64, 256, 512), (65, 128, 4096),
    (128, 4096, 1408), (129, 264, 64), (191, 128, 544), (192, 1000, 256), (193, 256, 224), (256, 512, 1024), (257, 264, 288),
    (300, 640, 4096), (384, 128, 128), (777, 392, 2080), (1025, 2056, 320), (40, 19000, 256), (2000, 4096, 512)])
def test_linear(fmt, M, N, K):
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=K ** -0.5).cuda(), fmt)
    _check(_rand(M, K, seed=2), w4, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 33, 200, 520])
def test_linear_epilogue(fmt, M):
    N, K = 264, 288
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=K ** -0.5).cuda(), fmt)
    x, bias, res = _rand(M, K, seed=2), _rand(N, seed=3), _rand(M, N, seed=4)
    _check(x, w4, fmt, bias=bias)
    _check(x, w4, fmt, act="gelu", bias=bias)
    _check(x, w4, fmt, residual=res)
    _check(x, w4, fmt, bias=bias, act="gelu", residual=res)


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_ranges_of_values(fmt):
    """Rows of very different sizes, zeros, scales that vanish; factors of a weight that are no powers of two."""
    K, N = 512, 136
    x = special_rows(K, seed=5)
    x[9] *= 1e-6       # (the largest numbers' products would pass bf16's range)
    x[4] *= 1e-6
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.05).cuda(), fmt)
    _check(x, w4, fmt)
    if fmt == "nvfp4":
        g = (0.01 + torch.rand(N, generator=torch.Generator().manual_seed(3))).cuda()
        _check(x, quant.Fp4Weight(w4.q, w4.scale, g, fmt), fmt)
        _check(x, quant.Fp4Weight(w4.q, w4.scale, None, fmt), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_every_code_and_scale(fmt):
    """Random bytes as codes, every finite scale byte: what the tensor core reads them as."""
    gen = torch.Generator().manual_seed(1)
    N, K = 256, 512
    q = torch.randint(0, 256, (N, K // 2), generator=gen, dtype=torch.uint8)
    blocks = K // quant.FP4_BLOCK[fmt]
    s = torch.arange(N * blocks).reshape(N, blocks) % 127 if fmt == "nvfp4" else \
        127 - 20 + torch.arange(N * blocks).reshape(N, blocks) % 41
    w4 = quant.Fp4Weight(q.cuda(), quant.tile_fp4_scales(s.to(torch.uint8)).cuda(), None, fmt)
    _check(_rand(48, K, seed=2), w4, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_rows_that_are_no_numbers_stay_alone(fmt):
    K, N = 256, 136
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), fmt)
    for M in (20, 300):
        x = _rand(M, K, seed=2)
        clean = ops.linear(x.cuda(), w4)
        x[3, 7], x[M - 1, 200] = float("inf"), float("nan")
        got = ops.linear(x.cuda(), w4)
        assert got[[3, M - 1]].isnan().all()
        keep = [i for i in range(M) if i not in (3, M - 1)]
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [5, 150, 400])
def test_linear_into_a_part_of_a_buffer(fmt, M):
    K, N = 320, 136
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), fmt)
    buf = torch.full((M + 3, N + 24), 5.0, dtype=torch.bfloat16, device="cuda")
    x, res = _rand(M, K, seed=2), _rand(M, 2 * N, seed=3)[:, :N]
    got = _check(x, w4, fmt, residual=res, out=buf[:M, 8:8 + N])
    assert got.data_ptr() == buf[:M, 8:].data_ptr()
    buf[:M, 8:8 + N] = 5.0
    assert bool((buf == 5).all())
    alone = ops.linear(x.cuda(), w4, residual=res.cuda())
    r = x.cuda().new_empty(M, 2 * N)[:, :N]
    r.copy_(res)
    assert torch.equal(ops.linear(x.cuda(), w4, residual=r), alone)
    assert torch.equal(ops.linear(x.cuda(), w4, residual=r, out=r), alone) and torch.equal(r, alone)     # in place


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_with_rows_of_a_weight(fmt):
    K = 192
    w4 = quant.quantize_weight_fp4(_rand(1000, K, seed=1, scale=0.1).cuda(), fmt)
    x = _rand(70, K, seed=2).cuda()
    whole = ops.linear(x, w4)
    for a, b in ((0, 128), (256, 520), (896, 1000)):
        assert torch.equal(ops.linear(x, w4[a:b]), whole[:, a:b])


@pytest.mark.parametrize("fmt", FORMATS)
def test_same_bits_every_time_and_for_every_batch(fmt):
    """A token's result does not depend on the run."""
    w4 = quant.quantize_weight_fp4(_rand(520, 1056, seed=1, scale=0.1).cuda(), fmt)
    x = ops.quant_fp4(_rand(400, 1056, seed=2).cuda(), fmt)
    first = ops.linear(x, w4)
    for _ in range(5):
        assert torch.equal(ops.linear(x, w4), first)


# ------------------------------------------------------------------------ experts
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("counts,even", [([1], False), ([6, 0, 1, 3], False), ([0, 0, 0, 2], False), ([127, 128, 129, 0, 40], False),
                                         ([300, 257, 0, 256, 511], False), ([300, 257, 0, 256, 511, 1], True),
                                         ([900, 640, 0, 700], True)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_experts(fmt, counts, even, act):
    E, N, K, n = len(counts), 288, 352, sum(counts)
    w = _rand(E, N, K, seed=1, scale=K ** -0.5)
    w4 = quant.quantize_weight_fp4(w.cuda(), fmt)
    _experts(fmt, counts, even, act, w4, _rand(n + 5, K, seed=2))


def _experts(fmt, counts, even, act, w4, x):
    n, N = sum(counts), w4.shape[1]
    r = routing_of(counts, "cuda", even)
    got = stream_ops.grouped_linear(x.cuda(), w4, r, act)
    ops.check_status()
    first = 0
    for e, c in enumerate(counts):
        if c:
            xd = oracle_rows(x[first:first + c], fmt).cuda()
            wd = oracle_values(w4.q[e], w4.scale[e], None if w4.row_scale is None else w4.row_scale[e], fmt).cuda()
            y = xd @ wd.t()
            bound = product_bound(xd, wd, y)
            if act is not None:
                g, u = (t.reshape(c, N // 2) for t in y.reshape(c, N // 32, 2, 16).unbind(2))
                eg, eu = (t.reshape(c, N // 2) for t in
                          (bound - 2.0 ** -8 * y.abs()).reshape(c, N // 32, 2, 16).unbind(2))
                y = stream_ops.Gate.of(act).join(g, u)
                # |d silu|, |d gelu| < 1.13, sigmoid's alpha up to 1.702; fast exponential and division: 2^-20
                bound = 2.0 ** -8 * y.abs() + 1.8 * (u.abs() + 1) * eg + (g.abs() + 0.3) * eu + \
                    2.0 ** -20 * (1 + g.abs()) * (1 + u.abs())
            bad = (got[first:first + c].double() - y).abs() > bound
            assert not bad.any(), (e, int(bad.sum()), bad.nonzero()[0].tolist())
        first += c
    return got


@pytest.mark.parametrize("act", ["gelu_tanh", stream_ops.Gate("clamped_swish", 1.5, 1.3)])
def test_experts_other_gates(act):
    counts, N, K = [40, 3, 130], 96, 256
    w4 = quant.quantize_weight_fp4(_rand(3, N, K, seed=1, scale=K ** -0.5).cuda(), "nvfp4")
    _experts("nvfp4", counts, False, act, w4, _rand(sum(counts), K, seed=2))


def test_experts_behind_the_router():
    """Router, experts' gate / up and down products and the rows that come back, as a layer runs them."""
    T, W, ff, E, top = 70, 256, 96, 8, 2
    x = _rand(T, W, seed=1)
    router = (0.1 * _rand(E, W, seed=2)).cuda()
    gate, up, down = (_rand(*s, seed=i, scale=0.06).cuda() for i, s in enumerate(((E, ff, W), (E, ff, W), (E, W, ff))))
    for fmt in FORMATS:
        w1 = quant.quantize_weight_fp4(stream_ops.interleave_gate_up(gate, up), fmt)
        w2 = quant.quantize_weight_fp4(down, fmt)
        routing, rows = stream_ops.route(x.cuda(), x.cuda(), router, torch.zeros(E, device="cuda"), top)
        h = stream_ops.grouped_linear(rows, w1, routing, "silu")
        y = stream_ops.grouped_linear(h, w2, routing)
        ops.check_status()
        ids, at = routing.ids.cpu(), routing.rows.cpu()
        v1, v2 = w1.dequantize().cpu().double(), w2.dequantize().cpu().double()
        xd, hd = oracle_rows(x, fmt), oracle_rows(h.cpu(), fmt)
        for t in range(0, T, 7):
            for k in range(top):
                e, r = int(ids[t, k]), int(at[t, k])
                v = (v1[e] @ xd[t]).reshape(-1, 2, 16)
                g, u = v[:, 0].flatten(), v[:, 1].flatten()
                assert torch.allclose(h[r].cpu().double(), g * torch.sigmoid(g) * u, rtol=2.0 ** -7, atol=1e-4)
                want = v2[e] @ hd[r]
                assert ((y[r].cpu().double() - want).abs() <= product_bound(hd[r][None], v2[e], want[None])[0]).all()


# ------------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 130])
def test_feed_forward_half(fmt, M):
    """Norm, gate / up, activation, down and residual; every step against the oracle on that step's own input."""
    H, I = 256, 352
    x, norm = _rand(M, H, seed=1).cuda(), (1 + 0.1 * _rand(H, seed=2)).cuda()
    w1 = quant.quantize_weight_fp4(_rand(2 * I, H, seed=3, scale=H ** -0.5).cuda(), fmt)
    w2 = quant.quantize_weight_fp4(_rand(H, I, seed=4, scale=I ** -0.5).cuda(), fmt)

    def run():
        y = ops.rmsnorm(x, norm, 1e-5, quant=fmt)
        gu = ops.linear(y, w1)
        h = ops.silu_mul_blocked(gu, quant=fmt)
        return y, gu, h, ops.linear(h, w2, residual=x)

    y, gu, h, out = run()
    d = lambda w: oracle_values(w.q, w.scale, w.row_scale, fmt)
    yd, hd = d_rows(y), d_rows(h)
    assert ((gu.cpu().double() - yd @ d(w1).t()).abs() <= product_bound(yd, d(w1), yd @ d(w1).t())).all()
    want = hd @ d(w2).t() + x.cpu().double()
    assert ((out.cpu().double() - want).abs() <= product_bound(hd, d(w2), want)).all()
    # captured and replayed with other inputs
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = run()
    for seed in (7, 8):
        x.copy_(_rand(M, H, seed=seed))
        g.replay()
        assert torch.equal(captured[3], run()[3])
    ops.check_status()


def d_rows(r):
    return oracle_values(r.q, r.scale, r.row_scale, r.fmt)


def test_two_streams():
    """Calls that overlap on two streams share nothing."""
    w = [quant.quantize_weight_fp4(_rand(2048, 1024, seed=i, scale=0.05).cuda(), "nvfp4") for i in range(2)]
    x = [_rand(m, 1024, seed=5 + i).cuda() for i, m in enumerate((48, 700))]
    want = [ops.linear(a, b) for a, b in zip(x, w)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear(x[i], w[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])
    ops.check_status()


def test_refusals():
    x, w4 = _rand(4, 64).cuda(), quant.quantize_weight_fp4(_rand(40, 64).cuda(), "nvfp4")
    e4 = quant.quantize_weight_fp4(_rand(2, 32, 64).cuda(), "nvfp4")
    r = routing_of([2, 2], "cuda")
    odd = quant.quantize_weight_fp4(_rand(36, 64).cuda(), "nvfp4")
    buf = torch.zeros(4, 44, dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: ops.linear(x, odd),
        lambda: ops.linear(x, w4, out=buf[:, :40]),
        lambda: ops.linear(x, w4, out=buf[:, 4:]),
        lambda: ops.linear(x, w4, residual=torch.zeros(40, 4, dtype=torch.bfloat16, device="cuda").t()),
        lambda: ops.linear(x.cpu(), w4),
        lambda: ops.linear(x, w4, bias=torch.zeros(40, dtype=torch.bfloat16)),
        lambda: ops.linear(ops.quant_fp4(x, "nvfp4", r), w4),
        lambda: ops.grouped_linear_fp4(ops.quant_fp4(x, "nvfp4"), e4, r),
        lambda: ops.grouped_linear_fp4(x, e4, routing_of([2, 1, 1], "cuda")),
        lambda: ops.rmsnorm(x, torch.ones(64, device="cuda"), 1e-5, quant="nvfp4"),
        lambda: ops.rmsnorm(x, x[0], 1e-5, residual=buf[:, :64], quant="nvfp4"),
        lambda: ops.rmsnorm(_rand(1, 16416).cuda(), _rand(16416).cuda(), 1e-5, quant="nvfp4"),
        lambda: ops.silu_mul_fp4(_rand(4, 40).cuda()),
        lambda: ops.dequant_fp4(w4, out=buf),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("case %d was not refused" % i)
    torch.cuda.synchronize()
    ops.check_status()


# ------------------------------------------------------------------------ calls at the edges of what is allowed
@pytest.mark.parametrize("fmt", FORMATS)
def test_lists_that_reach_beyond_the_rows(fmt):
    """A routing of more rows than there are: what is there is served, nothing beyond it is touched."""
    counts = [100, 60, 0, 90]
    w4 = quant.quantize_weight_fp4(_rand(4, 64, 96, seed=1, scale=0.1).cuda(), fmt)
    x = _rand(250, 96, seed=2)
    whole = stream_ops.grouped_linear(x.cuda(), w4, routing_of(counts, "cuda"))
    for even in (False, True):
        r = routing_of(counts, "cuda", even)
        for n in (250, 180, 110, 3):
            buf = torch.empty(n + 8, 96, dtype=torch.bfloat16, device="cuda")
            buf[:n] = x[:n].cuda()
            assert torch.equal(stream_ops.grouped_linear(buf[:n], w4, r), whole[:n])
            q = ops.quant_fp4(buf[:n], fmt, r)
            assert torch.equal(q.dequantize(), ops.quant_fp4(buf[:n], fmt).dequantize())
    r = routing_of(counts, "cuda")
    r.tiles[2:, 0] = 9                                  # no such expert: left out
    stream_ops.grouped_linear(x.cuda(), w4, r)
    ops.check_status()


@pytest.mark.parametrize("M", [3, 100, 300])
def test_factors_and_bias_on_any_boundary(M):
    N, K = 264, 2048
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.03).cuda(), "nvfp4")
    g = torch.cat([torch.zeros(1), 0.5 + torch.rand(N, generator=torch.Generator().manual_seed(3))]).cuda()[1:]
    bias = torch.cat([torch.zeros(1, dtype=torch.bfloat16), _rand(N, seed=4)]).cuda()[1:]
    assert g.data_ptr() % 8 and bias.data_ptr() % 4
    x = _rand(M, K, seed=2)
    got = ops.linear(x.cuda(), quant.Fp4Weight(w4.q, w4.scale, g, "nvfp4"), bias=bias)
    assert torch.equal(got, ops.linear(x.cuda(), quant.Fp4Weight(w4.q, w4.scale, g.clone(), "nvfp4"), bias=bias.clone()))
    _check(x, quant.Fp4Weight(w4.q, w4.scale, g, "nvfp4"), "nvfp4", bias=bias.cpu())


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_wider_than_the_quantisers_take(fmt):
    """Rows that were quantised elsewhere may be longer than 32768."""
    K, N, M = 33024, 16, 130
    x, w = (torch.randint(0, 256, (r, K // 2), generator=torch.Generator().manual_seed(r), dtype=torch.uint8) for r in (M, N))
    tile = lambda r: torch.full(quant.fp4_scale_tiles(r, K, fmt), 48 if fmt == "nvfp4" else 120, dtype=torch.uint8)
    xr, wr = quant.Fp4Rows(x, tile(M), None, fmt), quant.Fp4Weight(w, tile(N), None, fmt)
    xd, wd = (oracle_values(t.q, t.scale, None, fmt) for t in (xr, wr))
    got = ops.linear(quant.Fp4Rows(x.cuda(), tile(M).cuda(), None, fmt), quant.Fp4Weight(w.cuda(), tile(N).cuda(), None, fmt))
    y = xd @ wd.t()
    assert ((got.cpu().double() - y).abs() <= product_bound(xd, wd, y)).all()
    with pytest.raises(ValueError):
        ops.linear(torch.zeros(2, K, dtype=torch.bfloat16, device="cuda"), quant.Fp4Weight(w.cuda(), tile(N).cuda(), None, fmt))


def test_captured_calls_share_nothing():
    """Two graphs of the same layer replayed in turn, beside eager calls, on inputs that change."""
    w4 = quant.quantize_weight_fp4(_rand(520, 4096, seed=1, scale=0.02).cuda(), "nvfp4")
    xs = [_rand(m, 4096, seed=m).cuda() for m in (7, 140)]
    for x in xs:
        ops.linear(x, w4)
    torch.cuda.synchronize()
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear(x, w4)
        graphs.append((g, x, y))
    for step in range(4):
        for g, x, y in graphs:
            x.copy_(_rand(*x.shape, seed=10 * step + x.shape[0]))
            g.replay()
        for g, x, y in graphs:
            assert torch.equal(ops.linear(x, w4), y)
    ops.check_status()


def test_input_that_the_output_overwrites():
    w4 = quant.quantize_weight_fp4(_rand(256, 256, seed=1, scale=0.1).cuda(), "mxfp4")
    for M in (5, 300):
        x = _rand(M, 256, seed=2).cuda()
        want = ops.linear(x, w4)
        assert ops.linear(x, w4, out=x) is x and torch.equal(x, want)


def test_long_offsets():
    """Rows and weights whose elements lie more than 2^31 bytes apart."""
    K, N, M = 64, 136, 70
    big = torch.empty(M * (1 << 25), dtype=torch.bfloat16, device="cuda").view(M, 1 << 25)      # 4.7 GB
    x = big[:, :K]
    x.copy_(_rand(M, K, seed=2))
    w4 = quant.quantize_weight_fp4(_rand(N, K, seed=1, scale=0.1).cuda(), "nvfp4")
    out = big[:, 1024:1024 + N]
    assert torch.equal(ops.linear(x, w4, out=out), ops.linear(x.contiguous(), w4))
    res = big[:, 4096:4096 + N]
    res.copy_(_rand(M, N, seed=3))
    assert torch.equal(ops.linear(x, w4, residual=res), ops.linear(x.contiguous(), w4, residual=res.contiguous()))
    ops.check_status()


def test_refused_outputs_and_widths():
    x, w4 = _rand(4, 64).cuda(), quant.quantize_weight_fp4(_rand(40, 64).cuda(), "nvfp4")
    byte = dict(dtype=torch.uint8, device="cuda")
    none_x = quant.Fp4Rows(torch.empty(4, 0, **byte), torch.empty(1, 0, 512, **byte), None, "mxfp4")
    none_w = quant.Fp4Weight(torch.empty(40, 0, **byte), torch.empty(1, 0, 512, **byte), None, "mxfp4")
    one = torch.zeros(1, 40, dtype=torch.bfloat16, device="cuda")
    table = torch.ops.arcticinference_b200
    bad = [
        lambda: ops.linear(none_x, none_w),                       # no columns
        lambda: ops.linear(x, w4, out=one.expand(4, 40)),          # four rows in one place
        lambda: ops.linear(x, w4, out=torch.zeros(200, dtype=torch.bfloat16, device="cuda").as_strided((4, 40), (32, 1))),
        lambda: table.fp4_linear(x, None, None, None, w4.q, w4.scale, w4.row_scale, 0, None, None, 0,
                                 torch.zeros(1, dtype=torch.int32, device="cuda")),
        lambda: table.fp4_linear(x, None, None, None, w4.q, w4.scale, w4.row_scale, 0, None, None, 0,
                                 torch.zeros(8, dtype=torch.int32)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("case %d was not refused" % i)
    # (one row may have any stride; a residual may be one row for all)
    ops.linear(x[:1], w4, out=one)
    r = _rand(1, 40, seed=3).cuda()
    assert torch.equal(ops.linear(x, w4, residual=r.expand(4, 40)), ops.linear(x, w4, residual=r.repeat(4, 1)))
    torch.cuda.synchronize()
    ops.check_status()
