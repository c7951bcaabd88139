"""4-bit kernels where several of their mechanisms meet: K split inside clusters, rings that wrap, lists that say more than
they hold, factors at the ends of their range."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant

from fp4_util import FORMATS, oracle_rows, oracle_values, product_bound

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
