"""Operators on microscaled 4-bit numbers (nvfp4, mxfp4): quantisation of rows, alone and fused into the norm and the
activation that feed a linear layer, the way back, and the products of linear layers and experts.

CUDA tensors run ``csrc/quant_fp4.cu`` and ``csrc/gemm_fp4.cu``, on the stream that is current on the tensors' device; CPU
tensors the PyTorch restatements of :mod:`..models.quant`. Both operands of a product have the same format. What
cannot be served raises ``ValueError`` before anything is launched.
"""

from __future__ import annotations

import contextlib

import torch

from . import _ACT, launch_counter
from . import reference as ref


def _nat():
    from . import native
    return native


def _on(t: torch.Tensor):
    """The tensors' device as the current one for the launch."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _need(ok, what: str, *args) -> None:
    if not ok:
        raise ValueError(what % args if args else what)


def _same_device(t: torch.Tensor, *others) -> None:
    for o in others:
        if o is not None:
            _need(o.device == t.device, "tensors on %s and %s", t.device, o.device)


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """Rows of bf16 numbers that the kernels' 16-byte accesses can read."""
    _need(isinstance(x, torch.Tensor) and x.dim() == 2, "%s: a matrix", what)
    _need(x.dtype == torch.bfloat16, "%s: bf16, got %s", what, getattr(x, "dtype", type(x)))
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _empty(M: int, K: int, fmt: str, device, row_tiles=None):
    from ..models import quant
    tiles = quant.fp4_scale_tiles(M, K, fmt)
    if row_tiles is not None:
        tiles = (row_tiles,) + tiles[1:]
    return (torch.empty(M, K // 2, dtype=torch.uint8, device=device),
            torch.empty(tiles, dtype=torch.uint8, device=device),
            torch.empty(M, dtype=torch.float32, device=device) if fmt == "nvfp4" else None)


def _code(fmt: str) -> int:
    from ..models import quant
    return quant.FP4_FORMATS.index(quant.check_fp4_format(fmt))


def quant_fp4(x: torch.Tensor, fmt: str = "nvfp4", routing=None):
    """bf16 rows [M, K], K a multiple of 32 and at most 32768 -> ``Fp4Rows``. ``routing`` (a ``stream_ops.Routing``): the
    rows are sorted by expert and lie in its tiles; rows that no tile holds are left out."""
    from ..models import quant
    code = _code(fmt)
    x = _rows(x, "quant_fp4")
    M, K = x.shape
    _need(K % 32 == 0 and 0 < K <= 32768, "quant_fp4: K a multiple of 32 up to 32768, got %d", K)
    if not x.is_cuda:
        r = quant.quantize_fp4_ref(x, fmt)
        return r if routing is None else quant.Fp4Rows(r.q, r.scale, r.row_scale, fmt, routing)
    nat = _nat()
    tiles = num = None
    if routing is not None:
        tiles, num = routing.tiles, routing.num_tiles
        _same_device(x, tiles, num)
    q, scale, g = _empty(M, K, fmt, x.device, None if tiles is None else tiles.shape[0])
    if M:
        with _on(x):
            rc = nat.lib().ab200_quant_fp4(x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(),
                                           nat.ptr(g), M, K, code, nat.ptr(tiles), nat.ptr(num), nat.stream_ptr())
        nat.check(rc, "quant_fp4 M=%d K=%d" % (M, K))
        launch_counter.add(1)
    return quant.Fp4Rows(q, scale, g, fmt, routing)


def dequant_fp4(rows, out: torch.Tensor = None) -> torch.Tensor:
    """The bf16 numbers that ``rows`` (``Fp4Rows`` or ``Fp4Weight``) stand for, each rounded once; exact where the row
    factors are powers of two, as the quantisers' are. With a routing, rows that no tile holds are not written."""
    from ..models import quant
    shape, K = rows.shape, rows.shape[-1]
    if not rows.is_cuda:
        plain = rows if rows.routing is None else quant.Fp4Rows(rows.q, rows.scale, rows.row_scale, rows.fmt)
        y = quant.dequantize_fp4_ref(plain).to(torch.bfloat16)
        return y if out is None else out.copy_(y)
    nat = _nat()
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=rows.device)
    _need(out.shape == shape and out.dtype == torch.bfloat16 and out.is_contiguous(),
          "dequant_fp4: out is a contiguous bf16 tensor %s", tuple(shape))
    _same_device(rows.q, out, rows.scale, rows.row_scale)
    q, scale = rows.q, rows.scale
    if q.dim() == 3 or q.stride(1) != 1:
        q = q.contiguous()
    g = None if rows.row_scale is None else rows.row_scale.contiguous()
    R = rows.numel() // K if K else 0
    if R == 0 or K == 0:
        return out
    r = rows.routing
    with _on(q):
        rc = nat.lib().ab200_dequant_fp4(
            q.data_ptr(), q.stride(-2), scale.contiguous().data_ptr(), nat.ptr(g), out.data_ptr(), K, R, K, shape[-2],
            _code(rows.fmt), None if r is None else r.tiles.data_ptr(), None if r is None else r.num_tiles.data_ptr(),
            nat.stream_ptr())
    nat.check(rc, "dequant_fp4 M=%d K=%d" % (R, K))
    launch_counter.add(1)
    return out


def rmsnorm_fp4(x: torch.Tensor, weight: torch.Tensor, eps: float, residual=None, fmt: str = "nvfp4"):
    """RMSNorm(x (+ residual)) as ``Fp4Rows`` in one pass; ``residual`` (contiguous) is updated in place."""
    from ..models import quant
    code = _code(fmt)
    if not x.is_cuda:
        return quant.quantize_fp4_ref(ref.rmsnorm(x, weight, eps, residual), fmt)
    nat = _nat()
    x = _rows(x, "rmsnorm_fp4")
    M, K = x.shape
    _need(K % 32 == 0 and 0 < K <= 16384, "rmsnorm_fp4: a multiple of 32 columns up to 16384, got %d", K)
    _need(weight.dtype == torch.bfloat16 and weight.shape == (K,) and weight.is_contiguous() and
          weight.data_ptr() % 16 == 0, "rmsnorm_fp4: bf16 weight [%d]", K)
    _need(residual is None or residual.dtype == torch.bfloat16 and residual.shape == x.shape and
          residual.is_contiguous() and residual.data_ptr() % 16 == 0, "rmsnorm_fp4: contiguous bf16 residual %s",
          tuple(x.shape))
    _same_device(x, weight, residual)
    q, scale, g = _empty(M, K, fmt, x.device)
    if M:
        with _on(x):
            rc = nat.lib().ab200_rmsnorm_fp4(x.data_ptr(), x.stride(0), nat.ptr(residual), weight.data_ptr(),
                                             q.data_ptr(), q.stride(0), scale.data_ptr(), nat.ptr(g), M, K, float(eps),
                                             code, nat.stream_ptr())
        nat.check(rc, "rmsnorm_fp4 M=%d K=%d" % (M, K))
        launch_counter.add(1)
    return quant.Fp4Rows(q, scale, g, fmt)


def silu_mul_fp4(x: torch.Tensor, nblk: int = 1, fmt: str = "nvfp4"):
    """SiLU(gate) * up of rows of ``nblk`` (gate | up) blocks as ``Fp4Rows`` [M, width / 2] in one pass."""
    from ..models import quant
    code = _code(fmt)
    _need(x.dim() == 2 and nblk >= 1 and x.shape[1] % (2 * nblk) == 0, "silu_mul_fp4: %s in %d (gate | up) blocks",
          tuple(x.shape), nblk)
    if not x.is_cuda:
        return quant.quantize_fp4_ref(ref.silu_mul_blocked(x, nblk), fmt)
    nat = _nat()
    x = _rows(x, "silu_mul_fp4")
    M, K = x.shape[0], x.shape[1] // 2
    inter = K // nblk
    _need(K % 32 == 0 and inter % 8 == 0 and 0 < K <= 32768,
          "silu_mul_fp4: a multiple of 32 columns up to 32768 in blocks of a multiple of 8, got %d x %d", nblk, inter)
    q, scale, g = _empty(M, K, fmt, x.device)
    if M:
        with _on(x):
            rc = nat.lib().ab200_silu_mul_fp4(x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(),
                                              nat.ptr(g), M, inter, nblk, code, nat.stream_ptr())
        nat.check(rc, "silu_mul_fp4 M=%d K=%d" % (M, K))
        launch_counter.add(1)
    return quant.Fp4Rows(q, scale, g, fmt)


def _as_rows(x, fmt: str, routing=None):
    from ..models import quant
    if isinstance(x, quant.QuantAct):
        x = x.dequantize()
    if isinstance(x, torch.Tensor):
        return quant_fp4(x, fmt, routing)
    _need(isinstance(x, quant.Fp4Rows), "rows of a 4-bit product: bf16 or Fp4Rows, got %s", type(x).__name__)
    _need(x.fmt == fmt, "rows are %s and the weight is %s", x.fmt, fmt)
    _need(x.routing is routing, "rows were quantised for another routing")
    return x


def _launch(x, w, out, bias, residual, act, gate, routing):
    nat = _nat()
    M, K = x.shape
    E, N = (1 if w.q.dim() == 2 else w.q.shape[0]), w.shape[-2]
    _need(x.q.stride(1) == 1 and x.q.stride(0) % 16 == 0 and x.q.data_ptr() % 16 == 0 and w.q.stride(-1) == 1 and
          all(s % 16 == 0 for s in w.q.stride()[:-1]) and w.q.data_ptr() % 16 == 0,
          "4-bit product: rows of codes on 16-byte boundaries")
    _need(w.scale.is_contiguous() and x.scale.is_contiguous() and w.scale.data_ptr() % 16 == 0 and
          x.scale.data_ptr() % 16 == 0, "4-bit product: contiguous scale tiles")
    for f in (x.row_scale, w.row_scale):
        _need(f is None or f.is_contiguous(), "4-bit product: contiguous row factors")
    _same_device(x.q, w.q, x.scale, w.scale, x.row_scale, w.row_scale, out, bias, residual)
    tiles = num = None
    if routing is not None:
        tiles, num = routing.tiles, routing.num_tiles
        _same_device(x.q, tiles, num)
    with _on(x.q):
        rc = nat.lib().ab200_linear_fp4(
            x.q.data_ptr(), x.q.stride(0), x.scale.data_ptr(), nat.ptr(x.row_scale), w.q.data_ptr(), w.q.stride(-2),
            w.q.stride(0) if E > 1 else 0, w.scale.data_ptr(), nat.ptr(w.row_scale), out.data_ptr(), out.stride(0), M,
            N, K, E, _code(w.fmt), nat.ptr(bias), nat.ptr(residual), 0 if residual is None else residual.stride(0),
            _ACT[act], gate.code if gate else 0, gate.limit if gate else 0.0, gate.alpha if gate else 0.0,
            nat.ptr(tiles), nat.ptr(num), 0 if tiles is None else tiles.shape[0],
            nat.status_buffer(x.device).data_ptr(), nat.stream_ptr())
    nat.check(rc, "linear_fp4 M=%d N=%d K=%d" % (M, N, K))
    launch_counter.add(1)
    return out


def linear_fp4(x, w, bias=None, residual=None, act=None, out=None) -> torch.Tensor:
    """``out = act(x @ w.T + bias) + residual`` with both operands in 4 bits: ``x`` bf16 [M, K] (quantised here) or
    ``Fp4Rows``, ``w`` an ``Fp4Weight`` [N, K] with N a multiple of 8. Sums are fp32, the result is rounded once to bf16."""
    from ..models import quant
    _need(isinstance(w, quant.Fp4Weight) and w.q.dim() == 2, "linear_fp4: an Fp4Weight [N, K]")
    N, K = w.shape
    _need(len(x.shape) == 2 and x.shape[1] == K, "linear_fp4: rows %s and weight %s", tuple(x.shape), (N, K))
    _need(act in _ACT, "linear_fp4: activation %r", act)
    M = x.shape[0]
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, (M, N)), ("out", out, (M, N))):
        _need(t is None or t.dtype == torch.bfloat16 and tuple(t.shape) == shape, "linear_fp4: %s is bf16 %s", name,
              shape)
    x = _as_rows(x, w.fmt)
    if not w.is_cuda:
        y = quant.dequantize_fp4_ref(x) @ quant.dequantize_fp4_ref(w).t()
        if bias is not None:
            y = y + bias.float()
        if act == "gelu":
            y = torch.nn.functional.gelu(y)
        if residual is not None:
            y = y + residual.float()
        y = y.to(torch.bfloat16)
        return y if out is None else out.copy_(y)
    _need(N % 8 == 0, "linear_fp4: N a multiple of 8, got %d", N)
    for name, t in (("residual", residual), ("out", out)):
        _need(t is None or t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0,
              "linear_fp4: rows of %s on 16-byte boundaries", name)
    _need(bias is None or bias.is_contiguous(), "linear_fp4: a contiguous bias")
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=w.device)
    if M == 0 or N == 0:
        return out
    return _launch(x, w, out, bias, residual, act, None, None)


def grouped_linear_fp4(x, w, routing, act=None) -> torch.Tensor:
    """Rows sorted by expert [n, K] (bf16, or ``Fp4Rows`` quantised with ``routing``) times each row's expert matrix of ``w``
    [E, N, K], as :func:`..stream_ops.grouped_linear`. With ``act`` (a Gate) the matrices are interleaved gate / up
    ones, joined by it in the kernel. Rows that no tile of the routing holds are not written."""
    from ..models import quant
    from . import stream_ops
    act = None if act is None else stream_ops.Gate.of(act)
    _need(isinstance(w, quant.Fp4Weight) and w.q.dim() == 3, "grouped_linear_fp4: an Fp4Weight [E, N, K]")
    E, N, K = w.shape
    _need(len(x.shape) == 2 and x.shape[1] == K, "grouped_linear_fp4: rows %s and weights %s", tuple(x.shape),
          (E, N, K))
    _need(N % (32 if act else 8) == 0, "grouped_linear_fp4: N a multiple of %d, got %d", 32 if act else 8, N)
    if not w.is_cuda:
        x = quant.dequantize_fp4_ref(_as_rows(x, w.fmt, None if isinstance(x, torch.Tensor) else routing))
        m = quant.dequantize_fp4_ref(w)
        y = torch.cat([xe @ m[e].t() for e, xe in enumerate(x.split(routing.counts))])
        if act is not None:
            v = y.reshape(y.shape[0], N // 32, 2, 16)
            y = act.join(v[:, :, 0], v[:, :, 1]).reshape(y.shape[0], N // 2)
        return y.to(torch.bfloat16)
    _need(routing.num_experts == E, "grouped_linear_fp4: a routing of %d experts and %d matrices", routing.num_experts, E)
    x = _as_rows(x, w.fmt, routing)
    out = torch.empty(x.shape[0], N // 2 if act else N, dtype=torch.bfloat16, device=w.device)
    if x.shape[0] == 0 or N == 0:
        return out
    return _launch(x, w, out, None, None, None, act, routing)
