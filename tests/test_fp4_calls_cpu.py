"""Calls of the 4-bit operators that the documentation allows or refuses, without a GPU: the same as with one."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

import fp4_calls
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


def _all_refused(calls):
    taken = {}
    for name, f in calls.items():
        try:
            f()
            taken[name] = "not refused"
        except ValueError:
            pass
        except Exception as e:          # noqa: BLE001 (which one is the answer)
            taken[name] = repr(e)[:90]
    assert not taken, taken


@pytest.mark.parametrize("fmt", FORMATS)
def test_refused_norms_and_activations(fmt):
    _all_refused(fp4_calls.norm_and_activation("cpu", fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_refused_products(fmt):
    _all_refused(fp4_calls.products("cpu", fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_beyond_a_routing_and_a_routing_beyond_the_rows(fmt):
    """As with the kernels: what a tile holds and is there is served."""
    w4 = quant.quantize_weight_fp4(_rand(3, 64, 96, seed=1, scale=0.1), fmt)
    x, r = _rand(12, 96, seed=2), routing_of([4, 0, 5], "cpu")
    whole = stream_ops.grouped_linear(x[:9], w4, r)
    got = stream_ops.grouped_linear(x, w4, r)
    assert got.shape == (12, 64) and torch.equal(got[:9], whole)
    assert torch.equal(stream_ops.grouped_linear(x[:6], w4, r), whole[:6])


def test_arguments_that_would_be_ignored():
    """A 4-bit layer splits K as it needs, and quantised rows have no place given beforehand."""
    x, w4 = _rand(4, 64), quant.quantize_weight_fp4(_rand(32, 64), "nvfp4")
    calls = {
        "splits": lambda: ops.linear(x, w4, force_splits=2),
        "out of the norm": lambda: ops.rmsnorm(x, _rand(64), 1e-5, out=torch.empty_like(x), quant="nvfp4"),
        "out of the activation": lambda: ops.silu_mul_blocked(x, out=_rand(4, 32), quant="mxfp4"),
    }
    _all_refused(calls)
    assert ops.linear(x, w4, force_splits=0).shape == (4, 32)


@pytest.mark.parametrize("fmt", FORMATS)
def test_residuals_that_overlap_the_output(fmt):
    _all_refused(fp4_calls.overlaps("cpu", fmt))
    for call, apart in fp4_calls.no_overlaps("cpu", fmt):
        want = apart()
        assert torch.equal(call(), want)
