"""What the 4-bit operators are measured on: quantisation to microscaled e2m1 numbers, linear layers and
expert products with both operands in that form, at the widths of the serving and layer benchmarks.

Four kinds of case:

    quant     rows to 4 bits and back: what a calibration or a check of an activation's error does
    linear    a linear layer called with bf16 rows: they are quantised, then multiplied
    mlp       the feed-forward half of a layer as a quantised model runs it: norm with quantisation,
              gate / up, activation with quantisation, down and the residual
    experts   rows sorted by expert through the experts' gate / up and down products

Formats: ``nvfp4``, blocks of 16 with an e4m3 scale and one power of two per row (a weight's row factor may be any
number); ``mxfp4``, blocks of 32 with a power of two each. Codes hold two values per byte, the even column
in the low half. Scales lie in tiles of 128 rows by four blocks, 512 bytes each: byte
(r % 32) * 16 + (r // 32) * 4 + b of a tile is the scale of row r and block b.

Activations are normal with a factor per column, as behind a norm whose weights differ; weights have the variance of
a random checkpoint. Sizes follow from a case's numbers alone.
"""

import math

import torch

own = False

HIDDEN, INTER, QKV, GATE_UP = 4096, 14336, 6144, 28672     # Llama-3.1-8B
T_WIDTH, T_FF, T_EXPERTS, T_TOP = 2048, 1408, 64, 6        # layer benchmark, moe-2048
EPS = 1e-5
BLOCK = {"nvfp4": 16, "mxfp4": 32}
PAIR_ROWS = 640      # rows per expert from which the router lists an even number of tiles each


def _quant(rows, width, fmt):
    return {"op": "quant", "rows": rows, "width": width, "fmt": fmt}


def _linear(rows, n, k, fmt, bias=False, residual=False):
    return {"op": "linear", "rows": rows, "n": n, "k": k, "fmt": fmt, "bias": bias, "residual": residual}


def _mlp(rows, hidden, inter, fmt):
    return {"op": "mlp", "rows": rows, "hidden": hidden, "inter": inter, "fmt": fmt}


def _experts(rows, experts, width, ff, fmt):
    return {"op": "experts", "rows": rows, "experts": experts, "width": width, "ff": ff, "fmt": fmt}


def listed():
    return [
        # one token's hidden state: latency
        {"name": "quant_one", **_quant(1, HIDDEN, "nvfp4")},
        # an odd batch behind the activation, the widest rows, powers of two as scales
        {"name": "quant_wide", **_quant(777, INTER, "mxfp4")},
        # a prefill step's hidden states
        {"name": "quant_prefill", **_quant(8192, HIDDEN, "nvfp4")},
        # one user, gate / up: the weights are the work
        {"name": "linear_one", **_linear(1, GATE_UP, HIDDEN, "nvfp4")},
        # a decode step of 128 requests, attention's output projection
        {"name": "linear_decode", **_linear(128, HIDDEN, HIDDEN, "nvfp4", residual=True)},
        # a chunk of a prompt beside decodes, with biases
        {"name": "linear_ragged", **_linear(777, QKV, HIDDEN, "mxfp4", bias=True)},
        # a prefill step's gate / up
        {"name": "linear_prefill", **_linear(8192, GATE_UP, HIDDEN, "nvfp4")},
        # a decode step's feed-forward
        {"name": "mlp_decode", **_mlp(128, HIDDEN, INTER, "nvfp4")},
        # a prefill step's
        {"name": "mlp_prefill", **_mlp(4096, HIDDEN, INTER, "nvfp4")},
        # one user: six experts of one row each
        {"name": "experts_one", **_experts(T_TOP, T_EXPERTS, T_WIDTH, T_FF, "nvfp4")},
        # a decode step of 128 requests: ragged groups of a dozen rows, some empty
        {"name": "experts_decode", **_experts(128 * T_TOP, T_EXPERTS, T_WIDTH, T_FF, "mxfp4")},
        # a prefill step of 8192 tokens
        {"name": "experts_prefill", **_experts(8192 * T_TOP, T_EXPERTS, T_WIDTH, T_FF, "nvfp4")},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "mlp", "experts"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    if kind == "quant":
        width = 32 * _log(rng, 2, INTER // 32)
        return _quant(_log(rng, 1, min(16384, 33000000 // width)), width, fmt)
    if kind == "linear":
        n, k = 8 * _log(rng, 16, GATE_UP // 8), 32 * _log(rng, 4, INTER // 32)
        return _linear(_log(rng, 1, min(8192, 700000000000 // (n * k))), n, k, fmt, rng.random() < 0.4, rng.random() < 0.4)
    if kind == "mlp":
        hidden, inter = 32 * _log(rng, 8, HIDDEN // 32), 32 * _log(rng, 16, INTER // 32)
        return _mlp(_log(rng, 1, 4096), hidden, inter, fmt)
    experts, width, ff = _log(rng, 4, 128), 32 * _log(rng, 8, T_WIDTH // 32), 32 * _log(rng, 8, T_FF // 32)
    return _experts(_log(rng, 1, 24000), experts, width, ff, fmt)


# ------------------------------------------------------------------------ the format, in 32 bits
def _e2m1(v):
    """Nearest e2m1 code of v, ties to the even code, saturated; the sign is bit 3."""
    a = v.abs()
    c = (a > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= border) if up else (a > border)
    return c + 8 * (v < 0).to(torch.uint8)


def _pow2(e):
    """2^e exactly, e >= -127."""
    return torch.where(e > -127, (e.int() + 127) << 23, torch.full_like(e, 1 << 22, dtype=torch.int32)).view(torch.float32)


def _quantise(x, fmt):
    """[.., K] -> codes [.., K] (one per byte), block scales' bytes [.., K / block], row factors [..] or None."""
    size = BLOCK[fmt]
    b = x.float().reshape(*x.shape[:-1], x.shape[-1] // size, size)
    top = b.abs().amax(-1)
    if fmt == "mxfp4":
        e = (torch.frexp(top).exponent - 3).clamp(min=-127)
        e = torch.where(top > 0, e, -127)
        codes = _e2m1(b * _pow2(-e).unsqueeze(-1))
        return codes.reshape(x.shape), (e + 127).to(torch.uint8), None
    most = top.amax(-1)
    m, e = torch.frexp(most)             # most = m 2^e, 1/2 <= m < 1; 2688 = 0.65625 * 2^12
    e = (e - 12 + (m > 0.65625).int()).clamp(min=-126)
    g = torch.where(most > 0, _pow2(e), torch.ones_like(most))
    over = 1.0 / g
    s = (top * over.unsqueeze(-1) / 6.0).to(torch.float8_e4m3fn)
    f = s.float().unsqueeze(-1)
    v = torch.where(f > 0, b * over[..., None, None] / f, torch.zeros_like(b))
    return _e2m1(v).reshape(x.shape), s.view(torch.uint8), g


def _values(codes):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    return table[codes.int()]


def _expand(codes, scales, rows, fmt):
    """The numbers that codes, scales and row factors stand for."""
    s = scales.view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else _pow2(scales.int() - 127)
    v = _values(codes).reshape(*scales.shape, BLOCK[fmt]) * s.unsqueeze(-1)
    v = v.reshape(codes.shape)
    return v if rows is None else v * rows.unsqueeze(-1)


def _round_trip(x, fmt):
    return _expand(*_quantise(x, fmt), fmt)


def _pack(codes):
    c = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 2, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _unpack(q):
    return torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], 2 * q.shape[-1])


def _tile(s):
    """Scale bytes [.., R, S] into tiles [.., ceil(R / 128), ceil(S / 4), 512]."""
    R, S = s.shape[-2:]
    p = torch.zeros(*s.shape[:-2], -(-R // 128) * 128, -(-S // 4) * 4, dtype=torch.uint8, device=s.device)
    p[..., :R, :S] = s
    p = p.reshape(*s.shape[:-2], p.shape[-2] // 128, 4, 32, p.shape[-1] // 4, 4)
    return p.movedim(-2, -4).transpose(-2, -3).reshape(*s.shape[:-2], -(-R // 128), -(-S // 4), 512)


def _untile(t, R, S):
    p = t.reshape(*t.shape[:-1], 32, 4, 4).transpose(-2, -3).movedim(-4, -2)
    return p.reshape(*t.shape[:-3], t.shape[-3] * 128, t.shape[-2] * 4)[..., :R, :S]


# ------------------------------------------------------------------------ inputs
def _rows(gen, rows, width):
    x = torch.randn(rows, width, generator=gen, device="cuda")
    return (x * torch.exp(0.5 * torch.randn(width, generator=gen, device="cuda"))).to(torch.bfloat16)


def _weight(gen, *shape):
    """A quantised weight as a program keeps it: packed codes, scale tiles, row factors."""
    w = (torch.randn(*shape[:-1], shape[-1], generator=gen, device="cuda") / math.sqrt(shape[-1])).to(torch.bfloat16)
    fmt = gen.fmt
    codes, scales, rows = _quantise(w, fmt)
    return {"q": _pack(codes).contiguous(), "scale": _tile(scales).contiguous(), "rows": rows}


class _Gen(torch.Generator):
    fmt = "nvfp4"


def expert_counts(rows, experts):
    """Rows of each expert: ragged, some empty where there are few, the same for equal numbers."""
    share = [math.exp(1.2 * math.sin(2.3 * e + 0.7)) for e in range(experts)]
    total, acc, cuts = sum(share), 0.0, []
    for s in share:
        acc += s
        cuts.append(int(round(rows * acc / total)))
    return [b - a for a, b in zip([0] + cuts[:-1], cuts)]


def _tiles(counts):
    """The router's list: (expert, first row, rows) of at most 128 rows each."""
    n, E = sum(counts), len(counts)
    even = n >= PAIR_ROWS * E
    out, first = [], 0
    for e, c in enumerate(counts):
        k = 0
        for r in range(0, c, 128):
            out.append((e, first + r, min(128, c - r), 0))
            k += 1
        if even and k % 2:
            out.append((e, first, 0, 0))
        first += c
    most = n // 128 + 2 * E if even else min(n, n // 128 + E)
    return out + [(0, 0, 0, 0)] * (most - len(out)), len(out), even


def prepare(case, seed):
    gen = _Gen(device="cuda")
    gen.manual_seed(seed)
    gen.fmt = case["fmt"]
    st = {"case": case}
    if case["op"] == "quant":
        st["x"] = _rows(gen, case["rows"], case["width"])
    elif case["op"] == "linear":
        st["x"] = _rows(gen, case["rows"], case["k"])
        st["w"] = _weight(gen, case["n"], case["k"])
        st["bias"] = torch.randn(case["n"], generator=gen, device="cuda").to(torch.bfloat16) if case["bias"] else None
        st["residual"] = _rows(gen, case["rows"], case["n"]) if case["residual"] else None
    elif case["op"] == "mlp":
        st["x"] = _rows(gen, case["rows"], case["hidden"])
        st["norm"] = (1 + 0.1 * torch.randn(case["hidden"], generator=gen, device="cuda")).to(torch.bfloat16)
        st["w"] = _weight(gen, 2 * case["inter"], case["hidden"])
        st["down"] = _weight(gen, case["hidden"], case["inter"])
    else:
        counts = expert_counts(case["rows"], case["experts"])
        tiles, used, even = _tiles(counts)
        st["x"] = _rows(gen, case["rows"], case["width"])
        # gate and up rows alternate in blocks of 16
        st["w"] = _weight(gen, case["experts"], 2 * case["ff"], case["width"])
        st["down"] = _weight(gen, case["experts"], case["width"], case["ff"])
        st["tiles"] = torch.tensor(tiles, dtype=torch.int32, device="cuda")
        st["used"] = torch.tensor([used], dtype=torch.int32, device="cuda")
        st["even"] = even
        st["counts"] = torch.tensor(counts, device="cuda")
        st["most"] = max(counts)
    return st


# ------------------------------------------------------------------------ one pass
def _plain_weight(w, fmt):
    q = _unpack(w["q"])
    return _expand(q, _untile(w["scale"], q.shape[-2], q.shape[-1] // BLOCK[fmt]), w["rows"], fmt)


def _plain_linear(x, w, fmt, bias=None, residual=None):
    y = _round_trip(x, fmt) @ _plain_weight(w, fmt).t()
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(torch.bfloat16)


def _join(g, u):
    return (g / (1 + torch.exp(-g)) * u).to(torch.bfloat16)


def _plain_mlp(st, fmt):
    x = st["x"].float()
    y = (x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * st["norm"].float()).to(torch.bfloat16)
    gu = _plain_linear(y, st["w"], fmt).float()
    half = gu.shape[1] // 2
    return _plain_linear(_join(gu[:, :half], gu[:, half:]), st["down"], fmt, residual=st["x"])


def _plain_experts(st, fmt):
    """Every expert's rows padded to the longest group's: products of a batch."""
    x, counts, most = st["x"], st["counts"], st["most"]
    first = torch.cumsum(counts, 0) - counts
    expert = torch.repeat_interleave(torch.arange(counts.numel(), device="cuda"), counts, output_size=x.shape[0])
    place = expert * most + torch.arange(x.shape[0], device="cuda") - first[expert]

    def product(rows, w):
        v = _plain_weight(w, fmt)
        p = torch.zeros(counts.numel() * most, rows.shape[1], device="cuda")
        p[place] = _round_trip(rows, fmt)
        return torch.bmm(p.view(counts.numel(), most, -1), v.transpose(1, 2)).reshape(counts.numel() * most, -1)[place]

    gu = product(x, st["w"]).reshape(x.shape[0], -1, 2, 16)
    h = _join(gu[:, :, 0], gu[:, :, 1]).reshape(x.shape[0], -1)
    return product(h, st["down"]).to(torch.bfloat16)


def run(state):
    case = state["case"]
    fmt = case["fmt"]
    if own:
        from arcticinference_b200 import ops
        from arcticinference_b200.models.quant import Fp4Weight
        from arcticinference_b200.ops import stream_ops

        def weight(w):
            return Fp4Weight(w["q"], w["scale"], w["rows"], fmt)

        if case["op"] == "quant":
            return ops.dequant_fp4(ops.quant_fp4(state["x"], fmt))
        if case["op"] == "linear":
            return ops.linear(state["x"], weight(state["w"]), bias=state["bias"], residual=state["residual"])
        if case["op"] == "mlp":
            y = ops.rmsnorm(state["x"], state["norm"], EPS, quant=fmt)
            h = ops.silu_mul_blocked(ops.linear(y, weight(state["w"])), quant=fmt)
            return ops.linear(h, weight(state["down"]), residual=state["x"])
        routing = stream_ops.Routing(None, None, None, 1, case["experts"], state["tiles"], state["used"], even=state["even"])
        h = stream_ops.grouped_linear(state["x"], weight(state["w"]), routing, act="silu")
        return stream_ops.grouped_linear(h, weight(state["down"]), routing)
    if case["op"] == "quant":
        return _round_trip(state["x"], fmt).to(torch.bfloat16)
    if case["op"] == "linear":
        return _plain_linear(state["x"], state["w"], fmt, state["bias"], state["residual"])
    if case["op"] == "mlp":
        return _plain_mlp(state, fmt)
    return _plain_experts(state, fmt)


# ------------------------------------------------------------------------ 64 bits, from the definition
def _double_pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _log2_floor(t):
    return torch.frexp(t).exponent - 1


def _exact_rows(x, fmt):
    """The numbers that the rows' 4-bit form stands for, in 64 bits."""
    size = BLOCK[fmt]
    b = x.double().reshape(x.shape[0], -1, size)
    top = b.abs().amax(-1)
    tiny = torch.finfo(torch.float64).tiny
    if fmt == "mxfp4":
        step = _double_pow2((_log2_floor(top.clamp(min=tiny)) - 2).clamp(min=-127))
    else:
        most = top.amax(-1, keepdim=True)
        low = _log2_floor(most.clamp(min=2.0 ** -200) / 2688)
        g = _double_pow2((low + (most > 2688 * _double_pow2(low)).int()).clamp(min=-126))
        t = top / (6 * g)
        grain = _double_pow2(_log2_floor(t.clamp(min=tiny)).clamp(min=-6) - 3)
        step = torch.round(t / grain) * grain * g
    step = step.unsqueeze(-1)
    a = b.abs()
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    at = torch.zeros(b.shape, dtype=torch.int64, device=x.device)
    for i in range(7):
        border = (grid[i] + grid[i + 1]) / 2 * step       # exact: few bits times few bits
        at += ((a >= border) if i % 2 else (a > border)).long()
    v = torch.where(step > 0, grid[at] * step, torch.zeros_like(b))
    return (torch.sign(b) * v).reshape(x.shape)


def _exact_weight(w, fmt):
    N, half = w["q"].shape
    size = BLOCK[fmt]
    low, high = (w["q"] & 15).long(), (w["q"] >> 4).long()
    c = torch.stack([low, high], -1).reshape(N, 2 * half)
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e > 0, (1 + m / 2) * _double_pow2(e - 1), m / 2) * (1 - 2 * (c >> 3)).double()
    r, s = torch.arange(N, device=c.device), torch.arange(2 * half // size, device=c.device)
    at = (r // 128)[:, None] * w["scale"].shape[1] * 512 + (s // 4)[None] * 512 + (r % 32)[:, None] * 16 + (r % 128 // 32)[:, None] * 4 + (s % 4)[None]
    byte = w["scale"].reshape(-1)[at].long()
    if fmt == "mxfp4":
        scale = _double_pow2(byte - 127)
    else:
        e, m = byte >> 3, (byte & 7).double()
        scale = torch.where(e > 0, (1 + m / 8) * _double_pow2(e - 7), m / 8 * 2.0 ** -6)
    v = (v.reshape(N, -1, size) * scale.unsqueeze(-1)).reshape(N, 2 * half)
    return v if w["rows"] is None else v * w["rows"].double()[:, None]


def _exact_linear(x, w, fmt):
    return _exact_rows(x, fmt) @ _exact_weight(w, fmt).t()


def exact(case, seed):
    st = prepare(case, seed)
    fmt = case["fmt"]
    if case["op"] == "quant":
        return _exact_rows(st["x"], fmt)
    if case["op"] == "linear":
        y = _exact_linear(st["x"], st["w"], fmt)
        y = y if st["bias"] is None else y + st["bias"].double()
        return y if st["residual"] is None else y + st["residual"].double()
    # (the values between the products are rounded to bf16 by definition)
    if case["op"] == "mlp":
        x = st["x"].double()
        y = (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * st["norm"].double()).to(torch.bfloat16)
        g, u = _exact_linear(y, st["w"], fmt).to(torch.bfloat16).double().chunk(2, 1)
        return _exact_linear((g * torch.sigmoid(g) * u).to(torch.bfloat16), st["down"], fmt) + x
    out, first = [], 0
    for e, c in enumerate(st["counts"].tolist()):
        if c:
            pick = lambda w: {"q": w["q"][e], "scale": w["scale"][e], "rows": None if w["rows"] is None else w["rows"][e]}
            gu = _exact_linear(st["x"][first:first + c], pick(st["w"]), fmt).reshape(c, -1, 2, 16)
            h = (gu[:, :, 0] * torch.sigmoid(gu[:, :, 0]) * gu[:, :, 1]).to(torch.bfloat16).reshape(c, -1)
            out.append(_exact_linear(h, pick(st["down"]), fmt))
        first += c
    return torch.cat(out)


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    per = 0.5 + 1 / BLOCK[case["fmt"]]       # bytes of a quantised number
    rows = case["rows"]
    if case["op"] == "quant":
        return {"bytes": rows * case["width"] * (2 + per + 2), "flops": 0}
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": rows * k * 2 + n * k * per + 2 * rows * n * (2 if case["residual"] else 1), "flops": 2 * rows * n * k}
    if case["op"] == "mlp":
        h, i = case["hidden"], case["inter"]
        return {"bytes": 2 * rows * h * 2 + 3 * h * i * per, "flops": 6 * rows * h * i}
    used = sum(c > 0 for c in expert_counts(rows, case["experts"]))
    w, f = case["width"], case["ff"]
    return {"bytes": 2 * rows * w * 2 + 3 * used * w * f * per, "flops": 6 * rows * w * f}
