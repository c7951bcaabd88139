"""The 4-bit operators without a GPU: the PyTorch restatement against the 64-bit oracle, the layout of scales, the
products' composition and what is refused."""

import pytest
import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

from fp4_util import FORMATS, oracle_rows, oracle_values, product_bound, routing_of, special_rows


def _rand(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K", [32, 96, 224, 1024])
def test_rows_are_those_of_the_definition(fmt, K):
    x = torch.cat([special_rows(K), _rand(150, K)])
    r = ops.quant_fp4(x, fmt)
    want = oracle_rows(x, fmt)
    assert torch.equal(oracle_values(r.q, r.scale, r.row_scale, fmt), want)
    assert torch.equal(r.dequantize(), want.to(torch.bfloat16))          # (exact: six bits)
    assert r.shape == x.shape and (r.row_scale is None) == (fmt == "mxfp4")


@pytest.mark.parametrize("fmt", FORMATS)
def test_values_that_are_no_numbers(fmt):
    x = _rand(6, 128)
    x[1, 5], x[2, 70], x[3, 127] = float("nan"), float("inf"), float("-inf")
    y = ops.quant_fp4(x, fmt).dequantize()
    for row, at in ((1, 5), (2, 70), (3, 127)):
        lost = torch.arange(128) // 32 == at // 32 if fmt == "mxfp4" else torch.ones(128, dtype=torch.bool)
        assert torch.equal(y[row].isnan(), lost)
    assert not y[[0, 4, 5]].isnan().any()


@pytest.mark.parametrize("shape", [(1, 1), (128, 4), (129, 5), (300, 7), (3, 130, 6)])
def test_scale_tiles(shape):
    s = torch.randint(0, 256, shape, dtype=torch.uint8)
    t = quant.tile_fp4_scales(s)
    R, S = shape[-2:]
    assert t.shape == (*shape[:-2], -(-R // 128), -(-S // 4), 512)
    assert torch.equal(quant.untile_fp4_scales(t, R, S), s)
    r, b = R - 1, S - 1
    assert torch.equal(t[..., r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4], s[..., r, b])
    assert int(t.long().sum()) == int(s.long().sum())                   # zeros beyond the matrix


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_and_its_epilogue(fmt):
    M, N, K = 5, 24, 96
    x, w, bias, res = _rand(M, K), _rand(N, K, seed=1), _rand(N, seed=2), _rand(M, N, seed=3)
    w4 = quant.quantize_weight_fp4(w, fmt)
    xd, wd = oracle_rows(x, fmt), oracle_rows(w, fmt)
    y = xd @ wd.t() + bias.double()
    got = ops.linear(x, w4, bias=bias, act="gelu", residual=res)
    want = torch.nn.functional.gelu(y) + res.double()
    assert ((got.double() - want).abs() <= product_bound(xd, wd, want)).all()
    out = torch.empty(M, N, dtype=torch.bfloat16)
    assert ops.linear(ops.quant_fp4(x, fmt), w4, out=out) is out
    assert ((out.double() - xd @ wd.t()).abs() <= product_bound(xd, wd, xd @ wd.t())).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_norm_and_activation_give_the_rows_of_their_results(fmt):
    x, w, res = _rand(4, 64), _rand(64, seed=1), _rand(4, 64, seed=2)
    r2 = res.clone()
    a = ops.rmsnorm(x, w, 1e-5, residual=res, quant=fmt)
    b = ops.quant_fp4(ops.rmsnorm(x, w, 1e-5, residual=r2), fmt)
    assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale) and torch.equal(res, r2)
    gu = _rand(4, 256, seed=4)
    a = ops.silu_mul_blocked(gu, 2, quant=fmt)
    b = ops.quant_fp4(ops.silu_mul_blocked(gu, 2), fmt)
    assert torch.equal(a.q, b.q) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", [None, "silu", stream_ops.Gate("clamped_swish", 2.0, 1.5)])
def test_experts(fmt, act):
    counts, N, K = [3, 0, 5, 1], 64, 96
    x, w = _rand(9, K), _rand(4, N, K, seed=1, scale=0.2)
    w4 = quant.quantize_weight_fp4(w, fmt)
    assert w4.shape == (4, N, K)
    got = stream_ops.grouped_linear(x, w4, routing_of(counts, "cpu"), act)
    xd = oracle_rows(x, fmt).split(counts)
    y = torch.cat([xe @ oracle_rows(w[e], fmt).t() for e, xe in enumerate(xd)])
    if act is not None:
        v = y.reshape(9, 2, 2, 16)
        y = stream_ops.Gate.of(act).join(v[:, :, 0], v[:, :, 1]).reshape(9, N // 2)
    assert got.shape == y.shape and torch.allclose(got.double(), y, rtol=2.0 ** -7, atol=1e-5)


def test_slices_of_a_weight():
    w = _rand(300, 64)
    w4 = quant.quantize_weight_fp4(w, "nvfp4")
    for a, b in ((0, 8), (128, 300), (256, 264), (0, 300)):
        s = w4[a:b]
        assert torch.equal(s.dequantize(), w4.dequantize()[a:b]) and s.shape == (b - a, 64)
    for bad in (slice(8, 16), slice(0, 128, 2), 5, (slice(0, 128), slice(0, 32))):
        with pytest.raises(ValueError):
            w4[bad]


def test_weights_are_overwritten_in_place():
    a, b = _rand(40, 64), _rand(40, 64, seed=9)
    for fmt in FORMATS:
        w = quant.quantize_weight_fp4(a, fmt)
        at = (w.q.data_ptr(), w.scale.data_ptr())
        w.requantize_from(b.float())
        assert (w.q.data_ptr(), w.scale.data_ptr()) == at
        assert torch.equal(w.dequantize(), quant.quantize_weight_fp4(b, fmt).dequantize())


def test_refusals():
    x, w4 = _rand(4, 64), quant.quantize_weight_fp4(_rand(32, 64), "nvfp4")
    e4 = quant.quantize_weight_fp4(_rand(2, 32, 64), "nvfp4")
    bad = [
        lambda: ops.quant_fp4(x, "fp4"),
        lambda: ops.quant_fp4(x.float()),
        lambda: ops.quant_fp4(_rand(4, 48)),
        lambda: ops.quant_fp4(_rand(4, 4, 64)),
        lambda: ops.quant_fp4(_rand(1, 32800)),
        lambda: ops.silu_mul_fp4(_rand(4, 66), 4),
        lambda: ops.linear(_rand(4, 96), w4),
        lambda: ops.linear(x, w4, act="relu"),
        lambda: ops.linear(x, w4, bias=_rand(31)),
        lambda: ops.linear(x, w4, residual=_rand(4, 32).float()),
        lambda: ops.linear(x, w4, out=torch.empty(4, 31, dtype=torch.bfloat16)),
        lambda: ops.linear(ops.quant_fp4(x, "mxfp4"), w4),
        lambda: ops.linear(x, w4, sync=object()),
        lambda: ops.linear_fp4(x, e4),
        lambda: ops.grouped_linear_fp4(x, w4, routing_of([2, 2], "cpu")),
        lambda: ops.grouped_linear_fp4(_rand(4, 96), e4, routing_of([2, 2], "cpu")),
        lambda: ops.grouped_linear_fp4(x, quant.quantize_weight_fp4(_rand(2, 48, 64), "nvfp4"),
                                       routing_of([2, 2], "cpu"), "silu"),
        lambda: quant.quantize_weight_fp4(_rand(4, 40), "nvfp4"),
        lambda: quant.Fp4Weight(w4.q, w4.scale[:, :0], w4.row_scale, "nvfp4"),
        lambda: quant.Fp4Weight(w4.q, w4.scale, w4.row_scale[:3], "nvfp4"),
        lambda: quant.Fp4Weight(w4.q.float(), w4.scale, w4.row_scale, "nvfp4"),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("case %d was not refused" % i)


def test_no_rows():
    w4 = quant.quantize_weight_fp4(_rand(32, 64), "mxfp4")
    x = torch.empty(0, 64, dtype=torch.bfloat16)
    assert ops.linear(x, w4).shape == (0, 32) and ops.quant_fp4(x, "nvfp4").dequantize().shape == (0, 64)


def test_products_without_columns_are_refused():
    scale = torch.empty(1, 0, 512, dtype=torch.uint8)
    x = quant.Fp4Rows(torch.empty(4, 0, dtype=torch.uint8), scale, None, "mxfp4")
    w = quant.Fp4Weight(torch.empty(40, 0, dtype=torch.uint8), scale, None, "mxfp4")
    with pytest.raises(ValueError):
        ops.linear(x, w)
