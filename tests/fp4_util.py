"""64-bit oracle of the 4-bit operators, written from the formats' definitions."""

import torch

FORMATS = ("nvfp4", "mxfp4")
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def floor_log2(t):
    return torch.frexp(t).exponent - 1


def oracle_rows(x, fmt):
    """The numbers that the rows' 4-bit form stands for, fp64 on the CPU; finite rows."""
    x = x.detach().cpu().double()
    size = 16 if fmt == "nvfp4" else 32
    b = x.reshape(x.shape[0], -1, size)
    top = b.abs().amax(-1)
    low = 2.0 ** -300
    if fmt == "mxfp4":
        step = pow2((floor_log2(top.clamp(min=low)) - 2).clamp(min=-127))
    else:
        most = top.amax(-1, keepdim=True)
        e = floor_log2(most.clamp(min=low) / 2688)
        g = pow2((e + (most > 2688 * pow2(e)).int()).clamp(min=-126))
        t = top / (6 * g)
        grain = pow2(floor_log2(t.clamp(min=low)).clamp(min=-6) - 3)
        step = torch.round(t / grain) * grain * g          # to the nearest e4m3, ties to even
    step = step.unsqueeze(-1)
    q = torch.where(step > 0, b.abs() / step, torch.zeros_like(b))
    lower = torch.searchsorted(GRID, q.clamp(max=6.0).contiguous(), right=True).sub(1).clamp(max=6)
    mid = (GRID[lower] + GRID[lower + 1]) / 2
    up = (q > mid) | ((q == mid) & (lower % 2 == 1))
    return (torch.sign(b) * GRID[lower + up.long()] * step).reshape(x.shape)


def oracle_values(q, scale, row_scale, fmt):
    """fp64 numbers of packed codes [N, K / 2] and scale tiles."""
    q, scale = q.cpu(), scale.cpu()
    N, half = q.shape
    c = torch.stack([q & 15, q >> 4], -1).reshape(N, 2 * half).long()
    v = GRID[c & 7] * (1 - 2 * (c >> 3)).double()
    size = 16 if fmt == "nvfp4" else 32
    r, s = torch.arange(N)[:, None], torch.arange(2 * half // size)[None]
    byte = scale[r // 128, s // 4, r % 32 * 16 + r % 128 // 32 * 4 + s % 4].long()
    if fmt == "mxfp4":
        f = pow2(byte - 127)
    else:
        e, m = byte >> 3, (byte & 7).double()
        f = torch.where(e > 0, (1 + m / 8) * pow2(e - 7), m / 8 * 2.0 ** -6)
    v = (v.reshape(N, -1, size) * f.unsqueeze(-1)).reshape(N, 2 * half)
    return v if row_scale is None else v * row_scale.cpu().double()[:, None]


def product_bound(x, w, y):
    """How far a bf16 product may be from ``y`` = x @ w.T (+ what is added): half a bf16 step, and fp32 sums. The
    products of a block are exact and 16 of them are added at a time; every addition is off by at most one step of
    the sum's size (2^-23, chopped), and no partial sum is larger than the sum of magnitudes."""
    mag = x.abs() @ w.abs().t()
    return 2.0 ** -8 * y.abs() + (x.shape[1] / 16 + 8) * 2.0 ** -23 * mag + 1e-30


def special_rows(K, seed=0):
    """bf16 rows at the formats' edges."""
    gen = torch.Generator().manual_seed(seed)
    x = 3 * torch.randn(24, K, generator=gen)
    x[1] = 0
    x[2] = -0.0
    x[3] *= 1e-38                                   # subnormal numbers among them
    x[4] *= 1e30
    x[5, : K // 2] = 0                              # blocks of zeros
    x[6] = torch.randint(-24, 25, (K,), generator=gen) * 0.25           # ties of e2m1
    x[7] = 0
    x[7, K - 1] = 2688.0
    x[8] = 6.0 * 2.0 ** torch.randint(-12, 9, (K,), generator=gen)
    x[9] = x[0] / x[0].abs().max() * 3.3e38
    x[10] = 2.0 ** -133
    x[11] = torch.where(torch.arange(K) % 16 == 3, 1.0, 2.0 ** -20)
    x[12, 0] = 1e9                                  # the other blocks' scales go to zero
    x[13] = 2689.0 * torch.sign(x[13])
    x[14] = 7.0                                     # beyond the last value after a power of two
    x[15] = 5.0 * torch.sign(x[15])
    x[16] = 4.25 * (1 + torch.arange(K) % 3)
    x[17] = 2.0 ** -126
    return x.to(torch.bfloat16)


def routing_of(counts, device, even=False, slack=3):
    """The router's list for given rows per expert (tiles that are not in use hold what was there)."""
    from arcticinference_b200.ops import stream_ops
    tiles, first = [], 0
    for e, c in enumerate(counts):
        k = 0
        for r in range(0, c, 128):
            tiles.append((e, first + r, min(128, c - r), 0))
            k += 1
        if even and k % 2:
            tiles.append((e, first, 0, 0))
        first += c
    used = len(tiles)
    tiles += [(7, 1 << 20, 99, 0)] * slack
    return stream_ops.Routing(None, None, None, 1, len(counts), torch.tensor(tiles, dtype=torch.int32, device=device),
                              torch.tensor([used], dtype=torch.int32, device=device), counts=list(counts), even=even)


def checked_linears(monkeypatch, fmt):
    """Every linear layer that a model calls from now on is held to the oracle on its own input. (Whole forward passes
    are not comparable: attention outputs that differ by one bf16 step in one place of ten move the logits of a small
    random model by 10 to 30 per cent, because a code that changes changes by a quarter of its value.) Returns the list
    of shapes that were checked."""
    from arcticinference_b200 import ops
    from arcticinference_b200.models.quant import Fp4Rows, Fp4Weight
    inner, seen = ops.linear, []

    def linear(x, w, *args, **kw):
        y = inner(x, w, *args, **kw)
        if isinstance(w, Fp4Weight):
            assert not args and set(kw) <= {"bias", "sync"} and kw.get("sync") is None
            xd = oracle_values(x.q, x.scale, x.row_scale, fmt) if isinstance(x, Fp4Rows) else oracle_rows(x, fmt)
            wd = oracle_values(w.q, w.scale, w.row_scale, fmt)
            want = xd @ wd.t()
            if kw.get("bias") is not None:
                want = want + kw["bias"].cpu().double()
            bad = (y.cpu().double() - want).abs() > product_bound(xd, wd, want) + 2.0 ** -23
            assert not bad.any(), (tuple(y.shape), bad.nonzero()[0].tolist())
            seen.append((type(x).__name__, tuple(y.shape)))
        return y

    monkeypatch.setattr(ops, "linear", linear)
    return seen
