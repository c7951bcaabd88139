"""Operators on microscaled 4-bit numbers (nvfp4, mxfp4): quantisation of rows, alone and fused into the norm and the
activation that feed a linear layer, the way back, and the products of linear layers and experts.

CUDA tensors run ``csrc/quant_fp4.cu`` and ``csrc/gemm_fp4.cu``, on the stream that is current on the tensors' device; CPU
tensors the PyTorch restatements of :mod:`..models.quant`. Both operands of a product have the same format. What
cannot be served raises ``ValueError`` before anything is launched.

The kernels are reached through ``torch.ops.arcticinference_b200.fp4_*`` (csrc/torch/torch_bindings.cpp), which checks,
allocates and launches: a linear layer of few tokens is two launches of a few microseconds, and the same work in Python
took 60 us a call.
"""

from __future__ import annotations

import torch

from . import _ACT, launch_counter
from . import reference as ref

_FORMATS = {"nvfp4": 0, "mxfp4": 1}
_table = None


class _Ops:
    """The dispatcher's entries (their default overloads, which need no search per call)."""

    def __init__(self):
        from .. import build
        from ..models import quant
        from . import native
        t = build.load_torch_ops()
        self.quant, self.rmsnorm, self.silu_mul = t.fp4_quant.default, t.fp4_rmsnorm.default, t.fp4_silu_mul.default
        self.dequant, self.dequant_out = t.fp4_dequant.default, t.fp4_dequant_out.default
        self.linear = t.fp4_linear.default
        self.linear_out, self.grouped = t.fp4_linear_out.default, t.fp4_grouped_linear.default
        self.status, self.rows = native.status_buffer, quant.Fp4Rows._of


def _ops() -> _Ops:
    global _table
    if _table is None:
        _table = _Ops()
    return _table


def _need(ok, what: str, *args) -> None:
    if not ok:
        raise ValueError(what % args if args else what)


def _code(fmt: str) -> int:
    code = _FORMATS.get(fmt)
    if code is None:
        raise ValueError("4-bit format %r: %s are there" % (fmt, " and ".join(_FORMATS)))
    return code


def _bf16_matrix(x, what: str) -> None:
    _need(isinstance(x, torch.Tensor) and x.dim() == 2 and x.dtype == torch.bfloat16, "%s: a bf16 matrix", what)


def _width(K: int, most: int, what: str) -> None:
    _need(K % 32 == 0 and 0 < K <= most, "%s: a multiple of 32 columns up to %d, got %d", what, most, K)


def quant_fp4(x: torch.Tensor, fmt: str = "nvfp4", routing=None):
    """bf16 rows [M, K], K a multiple of 32 and at most 32768 -> ``Fp4Rows``. ``routing`` (a ``stream_ops.Routing``): the
    rows are sorted by expert and lie in its tiles; rows that no tile holds are left out."""
    code = _code(fmt)
    if not x.is_cuda:
        from ..models import quant
        _bf16_matrix(x, "quant_fp4")
        _width(x.shape[1], 32768, "quant_fp4")
        r = quant.quantize_fp4_ref(x, fmt)
        return r if routing is None else quant.Fp4Rows(r.q, r.scale, r.row_scale, fmt, routing)
    o = _ops()
    q, scale, g = o.quant(x, code) if routing is None else o.quant(x, code, routing.tiles, routing.num_tiles)
    launch_counter.add(1)
    return o.rows(q, scale, None if code else g, fmt, routing)


def dequant_fp4(rows, out: torch.Tensor = None) -> torch.Tensor:
    """The bf16 numbers that ``rows`` (``Fp4Rows`` or ``Fp4Weight``) stand for: block scale times row factor and that times the
    code, each rounded to fp32, then to bf16. Exact where the factors are powers of two, as the quantisers' are. With a routing, rows that no tile holds are not written."""
    if not rows.is_cuda:
        from ..models import quant
        plain = rows if rows.routing is None else quant.Fp4Rows(rows.q, rows.scale, rows.row_scale, rows.fmt)
        _need(out is None or out.dtype == torch.bfloat16 and out.shape == rows.shape and out.is_contiguous(),
              "dequant_fp4: out is a contiguous bf16 tensor of the rows' shape")
        y = quant.dequantize_fp4_ref(plain).to(torch.bfloat16)
        return y if out is None else out.copy_(y)
    r, o = rows.routing, _ops()
    args = (rows.q, rows.scale, rows.row_scale, _FORMATS[rows.fmt], None if r is None else r.tiles,
            None if r is None else r.num_tiles)
    launch_counter.add(1)
    if out is None:
        return o.dequant(*args)
    o.dequant_out(*args, out)
    return out


def rmsnorm_fp4(x: torch.Tensor, weight: torch.Tensor, eps: float, residual=None, fmt: str = "nvfp4"):
    """RMSNorm(x (+ residual)) as ``Fp4Rows`` in one pass; ``residual`` (contiguous) is updated in place."""
    code = _code(fmt)
    if not x.is_cuda:
        from ..models import quant
        _bf16_matrix(x, "rmsnorm_fp4")
        _width(x.shape[1], 16384, "rmsnorm_fp4")
        for name, t, shape in (("weight", weight, x.shape[1:]), ("residual", residual, x.shape)):
            _need(t is None or t.dtype == torch.bfloat16 and t.shape == shape and t.is_contiguous(),
                  "rmsnorm_fp4: a contiguous bf16 %s %s", name, tuple(shape))
        return quant.quantize_fp4_ref(ref.rmsnorm(x, weight, eps, residual), fmt)
    o = _ops()
    q, scale, g = o.rmsnorm(x, weight, eps, residual, code)
    launch_counter.add(1)
    return o.rows(q, scale, None if code else g, fmt, None)


def silu_mul_fp4(x: torch.Tensor, nblk: int = 1, fmt: str = "nvfp4"):
    """SiLU(gate) * up of rows of ``nblk`` (gate | up) blocks as ``Fp4Rows`` [M, width / 2] in one pass."""
    code = _code(fmt)
    if not x.is_cuda:
        from ..models import quant
        _bf16_matrix(x, "silu_mul_fp4")
        _need(nblk >= 1 and x.shape[1] % (2 * nblk) == 0, "silu_mul_fp4: %s in %d (gate | up) blocks",
              tuple(x.shape), nblk)
        K = x.shape[1] // 2
        _width(K, 32768, "silu_mul_fp4")
        _need(K // nblk % 8 == 0, "silu_mul_fp4: blocks of a multiple of 8 columns, got %d", K // nblk)
        return quant.quantize_fp4_ref(ref.silu_mul_blocked(x, nblk), fmt)
    o = _ops()
    q, scale, g = o.silu_mul(x, nblk, code)
    launch_counter.add(1)
    return o.rows(q, scale, None if code else g, fmt, None)


def _operand(x, w, routing=None):
    """The rows of a product as the entries take them: (bf16,) or (None, codes, scales, factors)."""
    if isinstance(x, torch.Tensor):
        return x, None, None, None
    from ..models import quant
    if isinstance(x, quant.QuantAct):
        return x.dequantize(), None, None, None
    _need(isinstance(x, quant.Fp4Rows), "rows of a 4-bit product: bf16 or Fp4Rows, got %s", type(x).__name__)
    _need(x.fmt == w.fmt, "rows are %s and the weight is %s", x.fmt, w.fmt)
    _need(x.routing is routing, "rows were quantised for another routing")
    return None, x.q, x.scale, x.row_scale


def linear_fp4(x, w, bias=None, residual=None, act=None, out=None) -> torch.Tensor:
    """``out = act(x @ w.T + bias) + residual`` with both operands in 4 bits: ``x`` bf16 [M, K] (quantised here) or
    ``Fp4Rows``, ``w`` an ``Fp4Weight`` [N, K] with N a multiple of 8. Sums are fp32, the result is rounded once to bf16.
    ``out`` may be ``residual``, or has no element of it."""
    code = _ACT.get(act)
    _need(code is not None, "linear_fp4: activation %r", act)
    wq = getattr(w, "q", None)
    _need(wq is not None and wq.dim() == 2 and hasattr(w, "fmt"), "linear_fp4: an Fp4Weight [N, K]")
    if not wq.is_cuda:
        return _linear_ref(x, w, bias, residual, act, out)
    x, xq, xs, xg = _operand(x, w)
    o = _ops()
    launch_counter.add(1 if x is None else 2)
    status = o.status(wq.device)
    if out is None:
        return o.linear(x, xq, xs, xg, wq, w.scale, w.row_scale, _FORMATS[w.fmt], bias, residual, code, status)
    o.linear_out(x, xq, xs, xg, wq, w.scale, w.row_scale, _FORMATS[w.fmt], bias, residual, code, status, out)
    return out


def _lies(t, ok: bool, what: str) -> None:
    """What the kernels' 16-byte accesses need of a CPU tensor too."""
    _need(t.device.type == "cpu", "4-bit product: %s on %s beside tensors on the CPU", what, t.device)
    _need(ok, "4-bit product: %s: rows on 16-byte boundaries", what)


def _ref_operand(t, what: str) -> None:
    """Codes, scales and factors as the kernels read them."""
    _lies(t.q, t.q.stride(-1) == 1 and all(s % 16 == 0 for s in t.q.stride()[:-1]) and t.q.data_ptr() % 16 == 0, what)
    _lies(t.scale, t.scale.is_contiguous(), what + "' scales")
    if t.row_scale is not None:
        _lies(t.row_scale, t.row_scale.is_contiguous(), what + "' factors")


def _ref_rows(x, w, routing=None):
    """The numbers that the rows of a product stand for, fp32."""
    from ..models import quant
    K = w.shape[-1]
    _need(K > 0, "4-bit product: rows without columns")
    _need(len(x.shape) == 2 and x.shape[1] == K, "4-bit product: rows %s and weight %s", tuple(x.shape), tuple(w.shape))
    _ref_operand(w, "weight")
    rows = x
    x, q, scale, g = _operand(x, w, routing)
    if x is None:
        _ref_operand(rows, "rows")
        return quant.dequantize_fp4_ref(quant.Fp4Rows(q, scale, g, w.fmt))
    _lies(x, True, "rows")
    return quant.dequantize_fp4_ref(quant_fp4(x, w.fmt))


def _shares(a, b) -> bool:
    """Whether two matrices of bf16 rows share an element, other than all of them in the same places."""
    M, width = a.shape
    if M == 0 or width == 0:
        return False
    sa, sb = (a.stride(0), b.stride(0)) if M > 1 else (width, width)
    apart = (a.data_ptr() - b.data_ptr()) // 2
    if apart == 0 and sa == sb or apart >= (M - 1) * sb + width or -apart >= (M - 1) * sa + width:
        return False
    if sa != sb or sa < width:
        return True
    return apart % sa < width or sa - apart % sa < width      # columns of equal pitch, beside one another


def _linear_ref(x, w, bias, residual, act, out):
    from ..models import quant
    N = w.shape[0]
    v = _ref_rows(x, w)
    M = v.shape[0]
    _need(N % 8 == 0, "4-bit product: N a multiple of 8, got %d", N)
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, (M, N)), ("out", out, (M, N))):
        if t is not None:
            _need(t.dtype == torch.bfloat16 and tuple(t.shape) == shape, "linear_fp4: %s is bf16 %s", name, shape)
            _lies(t, t.is_contiguous() if name == "bias" else
                  t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0, name)
    _need(out is None or M <= 1 or out.stride(0) >= N, "4-bit product: rows of out overlap")
    _need(out is None or residual is None or not _shares(residual, out), "4-bit product: out overlaps residual")
    y = v @ quant.dequantize_fp4_ref(w).t()
    if bias is not None:
        y = y + bias.float()
    if act == "gelu":
        y = torch.nn.functional.gelu(y)
    if residual is not None:
        y = y + residual.float()
    y = y.to(torch.bfloat16)
    return y if out is None else out.copy_(y)


def grouped_linear_fp4(x, w, routing, act=None) -> torch.Tensor:
    """Rows sorted by expert [n, K] (bf16, or ``Fp4Rows`` quantised with ``routing``) times each row's expert matrix of ``w``
    [E, N, K], as :func:`..stream_ops.grouped_linear`. With ``act`` (a Gate) the matrices are interleaved gate / up
    ones, joined by it in the kernel. Rows that no tile of the routing holds are not written."""
    from . import stream_ops
    act = None if act is None else stream_ops.Gate.of(act)
    wq = getattr(w, "q", None)
    _need(wq is not None and wq.dim() == 3 and hasattr(w, "fmt"), "grouped_linear_fp4: an Fp4Weight [E, N, K]")
    _need(routing.num_experts == wq.shape[0], "grouped_linear_fp4: a routing of %d experts and %d matrices",
          routing.num_experts, wq.shape[0])
    if not wq.is_cuda:
        return _grouped_ref(x, w, routing, act)
    x, xq, xs, xg = _operand(x, w, routing)
    o = _ops()
    launch_counter.add(1 if x is None else 2)
    return o.grouped(x, xq, xs, xg, wq, w.scale, w.row_scale, _FORMATS[w.fmt], routing.tiles, routing.num_tiles,
                     routing.even, act.code if act else 0, act.limit if act else 0.0, act.alpha if act else 0.0, o.status(wq.device))


def _grouped_ref(x, w, routing, act):
    from ..models import quant
    N = w.shape[1]
    v = _ref_rows(x, w, routing)
    _need(N % (32 if act else 8) == 0, "grouped_linear_fp4: N a multiple of %d, got %d", 32 if act else 8, N)
    m = quant.dequantize_fp4_ref(w)
    y, first = v.new_zeros(v.shape[0], N), 0
    for e, count in enumerate(routing.counts):
        y[first:first + count] = v[first:first + count] @ m[e].t()
        first += count
    if act is not None:
        v = y.reshape(y.shape[0], N // 32, 2, 16)
        y = act.join(v[:, :, 0], v[:, :, 1]).reshape(y.shape[0], N // 2)
    return y.to(torch.bfloat16)
