"""Engines with 4-bit linears on the GPU: logits against the CPU engine, captured decode steps, programmatic launches,
sleep and wake-up."""

import os
import subprocess
import sys

import pytest
import torch

from arcticinference_b200 import LLM, SamplingParams, ops
from arcticinference_b200.config import EngineArgs, ModelConfig
from arcticinference_b200.engine.llm_engine import LLMEngine
from arcticinference_b200.models.loader import load_llama_state, random_llama_state
from arcticinference_b200.models.quant import quantize_model_fp4

from fp4_util import FORMATS, checked_linears

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _first_step(device, fmt, prompts):
    eng = LLMEngine.from_engine_args(EngineArgs(model="llama-tiny", num_gpu_blocks_override=64, block_size=16,
                                                max_model_len=512), device=device)
    m = eng.runner.model
    state = random_llama_state(ModelConfig.from_pretrained("llama-tiny"), 5, 0.05, "cpu", torch.bfloat16)
    load_llama_state(m, ((k, v.to(device)) for k, v in state))
    quantize_model_fp4(m, fmt)
    for p in prompts:
        eng.add_request(None, p, SamplingParams(temperature=0, max_tokens=2, ignore_eos=True))
    batch, _ = eng.runner.prepare(eng.scheduler.schedule())
    with torch.inference_mode():
        out = m.compute_logits(m.forward(batch, eng.runner.kv)).double().cpu()
    return out, m


@pytest.mark.parametrize("fmt", FORMATS)
def test_linears_of_a_step(fmt, monkeypatch):
    prompts = [[3, 9, 27, 81, 243, 5, 700], list(range(40, 340)), [8]]
    seen = checked_linears(monkeypatch, fmt)
    got, m = _first_step("cuda:0", fmt, prompts)
    ops.check_status()
    assert len(seen) == 4 * len(m.layers) and got.isfinite().all()
    want, n = _first_step("cpu", fmt, prompts)
    for a, b in zip(m.layers, n.layers):       # the same numbers, whoever has quantised them
        for w in ("wqkv", "wo", "wgu", "wdown"):
            assert torch.equal(getattr(a, w).dequantize().cpu(), getattr(b, w).dequantize())


@pytest.mark.parametrize("fmt", FORMATS)
def test_captured_steps_give_the_tokens_of_eager_ones(fmt):
    prompts = [{"prompt_token_ids": list(range(1, 200))}, {"prompt_token_ids": [5, 6, 7]}, {"prompt_token_ids": [9] * 60}]
    sp = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    got = []
    for eager in (False, True):
        llm = LLM(model="llama-small", device="cuda:0", max_model_len=1024, num_gpu_blocks_override=128,
                  quantization=fmt, enforce_eager=eager)
        got.append([o.outputs[0].token_ids for o in llm.generate(prompts, sp)])
        assert eager or llm.engine.runner.graph_replays > 0
        ops.check_status()
        del llm
    assert [t[0] for t in got[0]] == [t[0] for t in got[1]]
    same = sum(int(a == b) for x, y in zip(*got) for a, b in zip(x, y))
    assert same >= 0.75 * 36


def test_sleep_and_wake_up():
    llm = LLM(model="llama-small", device="cuda:0", max_model_len=512, num_gpu_blocks_override=64, quantization="nvfp4",
              enable_sleep_mode=True)
    sp = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    before = llm.generate([{"prompt_token_ids": [5, 6, 7]}], sp)[0].outputs[0].token_ids
    llm.sleep(level=2)
    assert llm.engine.runner.model.layers[0].wo.q is None
    llm.wake_up()
    assert llm.generate([{"prompt_token_ids": [5, 6, 7]}], sp)[0].outputs[0].token_ids == before


CHILD = '''
import dataclasses, sys
import numpy as np, torch
from arcticinference_b200 import ops
from arcticinference_b200.config import (PRESETS, CacheConfig, EngineConfig, ParallelConfig, SchedulerConfig)
from arcticinference_b200.engine.llm_engine import LLMEngine
from arcticinference_b200.engine.request import Request
from arcticinference_b200.engine.sampling_params import SamplingParams
from arcticinference_b200.engine.scheduler import ScheduledRequest, SchedulerOutput
from arcticinference_b200.models import quant
from arcticinference_b200.ops import stream_ops as st

out, rng = {}, np.random.default_rng(0)
for fmt in ("nvfp4", "mxfp4"):
    model = dataclasses.replace(PRESETS["llama-small"], quantization=fmt)
    engine = LLMEngine(EngineConfig(model=model, parallel=ParallelConfig(),
                                    cache=CacheConfig(block_size=64, num_gpu_blocks=96, enable_prefix_caching=False),
                                    scheduler=SchedulerConfig(max_model_len=1024, max_num_seqs=64),
                                    load_format="dummy", seed=0), device="cuda")
    reqs = []
    for i, n in enumerate((700, 301, 5, 64)):
        r = Request("r%d" % i, rng.integers(0, 32000, n + 8).tolist(), SamplingParams(temperature=0.0, ignore_eos=True))
        r.block_ids = list(range(1 + 16 * i, 17 + 16 * i))
        reqs.append((r, n))
    with torch.inference_mode():
        for t in range(4):
            step = SchedulerOutput()
            for r, n in reqs:
                at, new = (0, n) if t == 0 else (n + t - 1, 1)
                step.scheduled.append(ScheduledRequest(r, at, new, 0, True, want=[new - 1]))
                step.total_tokens += new
            out["%s step %d" % (fmt, t)] = engine.runner.score(step).cpu()
    assert engine.runner.graph_replays >= 3
    del engine
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    for T in (20, 3001):
        x, w, b = rand(T, 256).bfloat16(), rand(6, 256) * 0.1, torch.zeros(6, device="cuda")
        w1 = quant.quantize_weight_fp4(rand(6, 1024, 256).bfloat16() / 16, fmt)
        w2 = quant.quantize_weight_fp4(rand(6, 256, 512).bfloat16() / 22, fmt)
        r, rows = st.route(x, x, w.bfloat16(), b, 3)
        assert r.even == (T > 2000)
        for _ in range(3):      # back to back
            y = st.grouped_linear(st.grouped_linear(rows, w1, r, act="silu"), w2, r)
        out["%s experts %d" % (fmt, T)] = y[r.rows.long()].cpu()
ops.check_status()
torch.save(out, sys.argv[1])
'''


def test_programmatic_launches_change_no_bit(tmp_path):
    """Steps of 4-bit models, prompts and captured decodes, and routed experts with few and many rows."""
    got = []
    for i, flag in enumerate("101"):
        env = dict(os.environ, AB200_PDL=flag, ARCTIC_B200_NO_AUTOBUILD="1", PYTHONPATH=ROOT)
        path = str(tmp_path / str(i))
        run = subprocess.run([sys.executable, "-c", CHILD, path], env=env, capture_output=True, text=True, timeout=600)
        assert run.returncode == 0, run.stderr[-3000:]
        got.append(torch.load(path))
    for other in got[1:]:
        assert got[0].keys() == other.keys() and len(other) == 12
        assert not [k for k in other if not torch.equal(got[0][k], other[k])]
