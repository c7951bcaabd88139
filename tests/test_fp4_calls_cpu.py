"""Calls of the 4-bit operators that the documentation allows or refuses, without a GPU: the same as with one."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

from fp4_util import FORMATS, routing_of


def _rand(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_routing_of_no_tokens(fmt):
    w4 = quant.quantize_weight_fp4(_rand(4, 64, 96, scale=0.1), fmt)
    r = routing_of([0, 0, 0, 0], "cpu")
    x = torch.empty(0, 96, dtype=torch.bfloat16)
    assert stream_ops.grouped_linear(x, w4, r).shape == (0, 64)
    assert stream_ops.grouped_linear(ops.quant_fp4(x, fmt, r), w4, r, "silu").shape == (0, 32)
