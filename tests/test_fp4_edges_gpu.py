"""4-bit kernels where several of their mechanisms meet: K split inside clusters, rings that wrap, lists that say more than
they hold, factors at the ends of their range."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

from fp4_util import FORMATS, oracle_rows, oracle_values, product_bound, routing_of

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
