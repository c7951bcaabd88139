"""How the 4-bit products are launched and what the C entries refuse, without a GPU."""

import ctypes
import re
import subprocess

import pytest

from arcticinference_b200 import build

SM_SHARED, CTA_RESERVED = 228 * 1024, 1024
SMS = 148


def _entry(name, *args):
    fn = getattr(build.load_kernels(), name)
    fn.restype, fn.argtypes = ctypes.c_int, list(args)
    return fn


def _plan(M, N, K, fmt):
    P = ctypes.POINTER
    fn = _entry("ab200_linear_fp4_plan", ctypes.c_longlong, *[ctypes.c_int] * 4, P(ctypes.c_int), P(ctypes.c_int),
                P(ctypes.c_longlong))
    parts, columns, smem = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
    assert fn(M, N, K, fmt, SMS, parts, columns, smem) == 0
    return parts.value, columns.value, smem.value


@pytest.mark.parametrize("fmt", [0, 1])
def test_clusters_that_share_an_sm_both_get_their_tensor_memory(fmt):
    """CTAs of a cluster wait for one another with their tensor memory in hand, so all that fit on an SM by their shared
    memory (and there are at most two by their registers) fit into its 512 columns."""
    seen = set()
    for M in (1, 5, 16, 17, 32, 33, 64, 65, 100, 128):
        for N in (8, 128, 264, 520, 1024, 4096, 6144, 9472, 9480, 28672):
            for K in (32, 256, 1024, 2048, 2304, 4096, 8192, 14336, 32768):
                parts, columns, smem = _plan(M, N, K, fmt)
                assert 0 < smem <= 227 * 1024 and columns in (64, 128, 256, 512)
                assert parts * -(-N // 128) <= SMS or parts == 1
                if parts > 1:
                    seen.add(parts)
                    # (38 KB: the smallest CTA of the bf16 and fp8 clusters, which hold up to 128 columns)
                    together = min(2, SM_SHARED // (smem + CTA_RESERVED))
                    assert columns * together <= 512, (M, N, K)
                    assert columns + 128 <= 512 or smem + 38 * 1024 > SM_SHARED, (M, N, K)
    assert seen == {2, 4}


def _linear_fp4(M, N, K, gate, act=0, tiles=False):
    """The C entry's answer to a call with pointers that nothing reads before the checks are done."""
    P, L, I, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float
    fn = _entry("ab200_linear_fp4", P, L, P, P, P, L, L, P, P, P, L, L, I, I, I, I, P, P, L, I, I, F, F, P, P, I, I, P, P)
    room = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(room) + 255 & ~255
    return fn(at, K // 2, at, None, at, K // 2, 0, at, None, at, N, M, N, K, 1, 0, None, None, 0, act, gate, 0.0, 0.0,
              at if tiles else None, at if tiles else None, 0, 0, at, None)


@pytest.mark.parametrize("M", [1, 100, 129, 300, 5000])
@pytest.mark.parametrize("gate", [1, 2, 3])
def test_a_gate_without_a_list_is_refused(M, gate):
    """Only products of lists join gate and up: others would store N columns where out has N / 2."""
    assert _linear_fp4(M, 256, 512, gate) == -2


def test_only_quantisers_that_a_call_reaches_are_built():
    """Sources 0 (plain), 1 (norm), 2 (activation); vectors a thread; whether a warp has a row. A norm's rows are never a
    warp's: its sum needs the block."""
    lib = build.load_kernels()._name
    names = subprocess.run(["nm", "-C", lib], capture_output=True, text=True, check=True).stdout
    found = {tuple(t.strip() for t in m.split(",")) for m in re.findall(r"\bquant_fp4_kernel<([^<>]*)>\(", names)}
    found = {(int(a.split(")")[-1]), int(v), w) for a, _, v, w in found}
    want = {(1, v, "false") for v in (1, 2, 4, 8)} | {(s, v, "false") for s in (0, 2) for v in (2, 4, 8)} | \
        {(0, v, "true") for v in (2, 4, 8)} | {(2, v, "true") for v in (2, 4)}
    assert found == want, (found - want, want - found)
