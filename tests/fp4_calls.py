"""Calls of the 4-bit operators that are refused with ValueError, on the CPU and on the GPU alike."""

import torch

from arcticinference_b200 import ops
from arcticinference_b200.models import quant

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
