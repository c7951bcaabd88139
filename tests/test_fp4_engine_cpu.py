"""Engines with 4-bit linears on the CPU: what they compute, live weight updates, sleep, and what is refused."""

import dataclasses

import pytest
import torch

from arcticinference_b200 import LLM, SamplingParams
from arcticinference_b200.config import PRESETS, EngineArgs, ModelConfig
from arcticinference_b200.engine.llm_engine import LLMEngine
from arcticinference_b200.models.loader import load_llama_state, random_llama_state
from arcticinference_b200.models.quant import Fp4Weight, quantize_model_fp4

from fp4_util import FORMATS, checked_linears

KW = dict(num_gpu_blocks_override=64, block_size=16, max_model_len=128)


def _engine(model="llama-tiny", **kw):
    return LLMEngine.from_engine_args(EngineArgs(model=model, **KW, **kw), device="cpu")


def _logits(eng, prompts):
    for p in prompts:
        eng.add_request(None, p, SamplingParams(temperature=0, max_tokens=2, ignore_eos=True))
    batch, _ = eng.runner.prepare(eng.scheduler.schedule())
    with torch.inference_mode():
        return eng.runner.model.compute_logits(eng.runner.model.forward(batch, eng.runner.kv)).double()


def _greedy(eng, prompt=(3, 1, 4, 1, 5, 9, 2, 6)):
    eng.add_request("g", list(prompt), SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True))
    out = None
    while eng.has_unfinished_requests():
        for o in eng.step():
            out = o
    return list(out.outputs[0].token_ids)


@pytest.mark.parametrize("model", ["llama-tiny", "llama-tiny-swiftkv", "qwen2-tiny"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_linears_of_a_step(model, fmt, monkeypatch):
    """All four linears of every layer run on 4-bit weights, the norm and the activation hand them quantised rows."""
    eng = _engine(model, quantization=fmt)
    m = eng.runner.model
    assert all(isinstance(getattr(lw, n), Fp4Weight) for lw in m.layers for n in ("wqkv", "wo", "wgu", "wdown"))
    seen = checked_linears(monkeypatch, fmt)
    logits = _logits(eng, [[3, 9, 27, 81, 243, 5, 700, 12, 13], list(range(40, 90))])
    assert logits.isfinite().all()
    layers = m.cfg.num_hidden_layers
    assert len(seen) == 4 * layers + (1 if "swiftkv" in model else 0)
    assert sum(kind == "Fp4Rows" for kind, _ in seen) == 3 * layers      # o_proj (and the K/V of all later layers): bf16


@pytest.mark.parametrize("model", ["llama-tiny-swiftkv", "qwen2-tiny", "qwen3-tiny"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_other_families_generate(model, fmt):
    llm = LLM(model=model, device="cpu", quantization=fmt, **KW)
    out = llm.generate([{"prompt_token_ids": [1, 2, 3, 4]}, {"prompt_token_ids": list(range(30))}],
                       SamplingParams(temperature=0, max_tokens=6, ignore_eos=True))
    assert [len(o.outputs[0].token_ids) for o in out] == [6, 6]


@pytest.mark.parametrize("model,fmt", [("llama-tiny", "nvfp4"), ("llama-tiny", "mxfp4"), ("llama-tiny-swiftkv", "nvfp4")])
def test_weights_are_updated_in_place(model, fmt):
    import socket
    from arcticinference_b200.server.weight_sync import WeightSender
    from arcticinference_b200.server.weight_sync.receiver import engine_sync_weights
    eng = _engine(model, quantization=fmt)
    before, at = _greedy(eng), [getattr(lw, n).q.data_ptr() for lw in eng.runner.model.layers for n in ("wo", "wdown")]
    state = dict(random_llama_state(ModelConfig.from_pretrained(model), 77, 0.05, "cpu", torch.bfloat16))
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    sender = WeightSender(state, device="cpu")
    th = sender.start([{"master_addr": "127.0.0.1", "master_port": port, "replica_ids": [0]}], bucket_size=1 << 20,
                      timeout=60)
    res = engine_sync_weights(eng, {"master_addr": "127.0.0.1", "master_port": port, "timeout": 60})
    sender.join(th)
    assert res["incomplete_layers"] == []
    assert at == [getattr(lw, n).q.data_ptr() for lw in eng.runner.model.layers for n in ("wo", "wdown")]
    fresh = _engine(model)
    load_llama_state(fresh.runner.model, state.items())
    quantize_model_fp4(fresh.runner.model, fmt)
    after = _greedy(eng)
    assert after == _greedy(fresh) and after != before


def test_what_is_refused():
    for kw in ({"tensor_parallel_size": 2}, {"ulysses_sequence_parallel_size": 2}, {"pipeline_parallel_size": 2}):
        with pytest.raises(NotImplementedError):
            EngineArgs(model="llama-tiny", quantization="nvfp4", **KW, **kw).create_engine_config()
    with pytest.raises(ValueError):
        EngineArgs(model="llama-tiny", quantization="fp4", **KW).create_engine_config()
    with pytest.raises(NotImplementedError):
        dataclasses.replace(PRESETS["llama-tiny"], quantization="mxfp4", intermediate_size=520).validate()
    with pytest.raises(NotImplementedError):
        EngineArgs(model="taralix-tiny", quantization="nvfp4", **KW).create_engine_config()
    ns = EngineArgs.add_cli_args(__import__("argparse").ArgumentParser()).parse_args(["--quantization", "mxfp4"])
    assert ns.quantization == "mxfp4"
