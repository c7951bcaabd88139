"""Calls of the 4-bit operators that are refused with ValueError, on the CPU and on the GPU alike."""

import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops

from fp4_util import routing_of


def _rand(*shape, seed=0, device="cpu", scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16).to(device)


def norm_and_activation(device, fmt):
    r = lambda *s: _rand(*s, device=device)
    wide, flat = r(4, 128), r(64)
    return {
        "norm: width no multiple of 32": lambda: ops.rmsnorm(r(4, 40), r(40), 1e-5, quant=fmt),
        "norm: width above 16384": lambda: ops.rmsnorm(r(1, 16416), r(16416), 1e-5, quant=fmt),
        "norm: three dimensions": lambda: ops.rmsnorm(r(2, 2, 64), flat, 1e-5, quant=fmt),
        "norm: fp32 rows": lambda: ops.rmsnorm(r(4, 64).float(), flat, 1e-5, quant=fmt),
        "norm: fp32 weight": lambda: ops.rmsnorm(r(4, 64), flat.float(), 1e-5, quant=fmt),
        "norm: weight of another width": lambda: ops.rmsnorm(r(4, 64), r(32), 1e-5, quant=fmt),
        "norm: weight with a stride": lambda: ops.rmsnorm(r(4, 64), r(128)[::2], 1e-5, quant=fmt),
        "norm: residual with a stride": lambda: ops.rmsnorm(r(4, 64), flat, 1e-5, residual=wide[:, :64], quant=fmt),
        "norm: residual of another shape": lambda: ops.rmsnorm(r(4, 64), flat, 1e-5, residual=r(3, 64), quant=fmt),
        "norm: fp32 residual": lambda: ops.rmsnorm(r(4, 64), flat, 1e-5, residual=r(4, 64).float(), quant=fmt),
        "activation: width no multiple of 32": lambda: ops.silu_mul_blocked(r(4, 80), quant=fmt),
        "activation: width above 32768": lambda: ops.silu_mul_blocked(r(1, 2 * 32800), quant=fmt),
        "activation: blocks of 4 columns": lambda: ops.silu_mul_blocked(r(4, 64), 8, quant=fmt),
        "activation: no blocks": lambda: ops.silu_mul_blocked(r(4, 64), 0, quant=fmt),
        "activation: fp32 rows": lambda: ops.silu_mul_blocked(r(4, 128).float(), quant=fmt),
        "activation: three dimensions": lambda: ops.silu_mul_blocked(r(2, 2, 128), quant=fmt),
    }


def products(device, fmt):
    r = lambda *s: _rand(*s, device=device)
    w = lambda *s: quant.quantize_weight_fp4(r(*s), fmt)
    other = {"nvfp4": "mxfp4", "mxfp4": "nvfp4"}[fmt]
    x, w4, e4, list2 = r(4, 64), w(40, 64), w(2, 32, 64), routing_of([2, 2], device)
    q = ops.quant_fp4(x, fmt)
    lone, buf = r(1, 40), r(4, 48)
    scaled = quant.Fp4Weight(w4.q, w4.scale, torch.ones(80, device=device)[::2], fmt)
    apart = torch.zeros(2 * q.scale.numel(), dtype=torch.uint8, device=device).view(*q.scale.shape, 2)[..., 0]
    codes = torch.zeros(4, 40, dtype=torch.uint8, device=device)
    return {
        "36 features": lambda: ops.linear(x, w(36, 64)),
        "fp32 rows": lambda: ops.linear(x.float(), w4),
        "three dimensions": lambda: ops.linear(x[None], w4),
        "another width": lambda: ops.linear(r(4, 96), w4),
        "rows of the other format": lambda: ops.linear(ops.quant_fp4(x, other), w4),
        "rows above 32768": lambda: ops.linear(r(1, 32800), quant.Fp4Weight(
            torch.zeros(8, 16400, dtype=torch.uint8, device=device),
            torch.zeros(quant.fp4_scale_tiles(8, 32800, fmt), dtype=torch.uint8, device=device), None, fmt)),
        "bias of another length": lambda: ops.linear(x, w4, bias=r(32)),
        "fp32 bias": lambda: ops.linear(x, w4, bias=r(40).float()),
        "bias with a stride": lambda: ops.linear(x, w4, bias=r(80)[::2]),
        "fp32 residual": lambda: ops.linear(x, w4, residual=r(4, 40).float()),
        "residual of fewer rows": lambda: ops.linear(x, w4, residual=r(3, 40)),
        "residual across": lambda: ops.linear(x, w4, residual=r(40, 4).t()),
        "out of another width": lambda: ops.linear(x, w4, out=r(4, 32)),
        "out with rows 44 apart": lambda: ops.linear(x, w4, out=r(4, 44)[:, :40]),
        "out off 16 bytes": lambda: ops.linear(x, w4, out=buf[:, 4:44]),
        "out of one row": lambda: ops.linear(x, w4, out=lone.expand(4, 40)),
        "out with rows that overlap": lambda: ops.linear(x, w4, out=r(200).as_strided((4, 40), (32, 1))),
        "activation": lambda: ops.linear(x, w4, act="relu"),
        "factors with a stride": lambda: ops.linear(x, scaled),
        "scales with a stride": lambda: ops.linear(quant.Fp4Rows(q.q, apart, q.row_scale, fmt), w4),
        "codes off 16 bytes": lambda: ops.linear(quant.Fp4Rows(codes[:, 8:], q.scale, q.row_scale, fmt), w4),
        "experts for a layer": lambda: ops.linear(x, e4),
        "rows of a routing for a layer": lambda: ops.linear(ops.quant_fp4(x, fmt, list2), w4),
        "a layer for experts": lambda: stream_ops.grouped_linear(x, w4, list2),
        "a routing of three experts": lambda: stream_ops.grouped_linear(x, e4, routing_of([2, 1, 1], device)),
        "rows without the routing": lambda: stream_ops.grouped_linear(q, e4, list2),
        "rows of another routing": lambda: stream_ops.grouped_linear(ops.quant_fp4(x, fmt, routing_of([2, 2], device)),
                                                                     e4, list2),
        "experts of another width": lambda: stream_ops.grouped_linear(r(4, 96), e4, list2),
        "experts: 36 features": lambda: stream_ops.grouped_linear(x, w(2, 36, 64), list2),
        "experts: 48 gate and up rows": lambda: stream_ops.grouped_linear(x, w(2, 48, 64), list2, "silu"),
        "expansion into fp32": lambda: ops.dequant_fp4(q, out=torch.empty(4, 64, device=device)),
        "expansion into another shape": lambda: ops.dequant_fp4(q, out=r(4, 96)),
        "expansion into a part of a buffer": lambda: ops.dequant_fp4(q, out=r(4, 128)[:, :64]),
    }


def overlaps(device, fmt):
    """A residual that shares elements with the output, but not all of them in the same places."""
    r = lambda *s: _rand(*s, device=device)
    w4, x, buf = quant.quantize_weight_fp4(r(40, 64), fmt), r(4, 64), r(6, 96)
    long = r(400)
    return {
        "a row above": lambda: ops.linear(x, w4, residual=buf[:4, :40], out=buf[1:5, :40]),
        "eight columns on": lambda: ops.linear(x, w4, residual=buf[:4, :40], out=buf[:4, 8:48]),
        "another distance of rows": lambda: ops.linear(x, w4, residual=long.as_strided((4, 40), (40, 1)),
                                                       out=long.as_strided((4, 40), (48, 1))),
        "one row for all, in the output": lambda: ops.linear(x, w4, residual=buf[:1, :40].expand(4, 40), out=buf[:4, :40]),
    }


def no_overlaps(device, fmt):
    """(call, the same with a residual of its own): parts of one buffer that share nothing, and the output itself."""
    r = lambda *s: _rand(*s, device=device)
    w4, x = quant.quantize_weight_fp4(r(40, 64), fmt), r(4, 64)
    out = []
    for res, to in ((lambda b: b[:4, :40], lambda b: b[:4, 48:88]), (lambda b: b[:4, 48:88], lambda b: b[:4, :40]),
                    (lambda b: b[:4, :40], lambda b: b[4:8, :40]), (lambda b: b[:4, 8:48], lambda b: b[:4, 8:48]),
                    (lambda b: b[4:5, :40].expand(4, 40), lambda b: b[:4, :40])):
        buf = r(9, 96)
        out.append((lambda b=buf, f=res, g=to: ops.linear(x, w4, residual=f(b), out=g(b)),
                    lambda b=buf.clone(), f=res: ops.linear(x, w4, residual=f(b).contiguous())))
    return out
