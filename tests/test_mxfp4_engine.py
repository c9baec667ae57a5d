"""
The engine with weights, and the rows they multiply, in microscaled 4-bit floating point: against the plain implementation over weights
that have been rounded the same way, replayed from CUDA graphs and not, and through the command line.
"""

from __future__ import annotations

import json
import subprocess
import sys

import pytest
import torch

import mxfp4_plain
import plain_llama as plain
import replay_util as ru
from tiny_configs import PAGE_A, PAGE_B, TINY_A, TINY_B

PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")
RAW, PAGES = {"a": TINY_A, "b": TINY_B}, {"a": PAGE_A, "b": PAGE_B}


def test_formats_that_are_refused():
    from tinyserve_llm_b200.engine.loading import check_formats
    check_formats(None, None, torch.float32)
    check_formats("mxfp4", "mxfp4", torch.bfloat16)
    for weights, rows, dtype in (("fp8", None, torch.bfloat16), ("mxfp4", "int4", torch.bfloat16), ("mxfp4", None, torch.float32),
                                 (None, "mxfp4", torch.bfloat16)):
        with pytest.raises(ValueError):
            check_formats(weights, rows, dtype)


def rounded_tensors(folder):
    cfg, tensors = plain.read_model_folder(folder)
    out = {}
    for name, t in tensors.items():
        if any(f"{p}.weight" in name for p in PROJECTIONS):
            t = torch.from_numpy(mxfp4_plain.rounded(t.double().numpy())).to(t.dtype)
        out[name] = t
    return cfg, out


def engine_logits(folder, page, ids, cut, formats, graphs=True):
    """Logits of every position: the first `cut` tokens as one prompt portion, the rest one by one."""
    from tinyserve_llm_b200.engine.loading import build_cache, load_model
    from tinyserve_llm_b200.engine.step import StepEntry, StepRunner
    model = load_model(folder, "bfloat16", "cuda", **formats)
    _, manager, storage = build_cache(model, page, 32, caching=False)
    runner = StepRunner(model, manager, storage, cuda_graphs=graphs)
    assert manager.admit(0, ids[:cut])
    rows = [runner.step([StepEntry(0, ids[:cut], list(range(cut)))]).cpu().clone()]
    manager.commit(0, cut)
    for token in ids[cut:]:
        manager.extend(0, [token])
        rows.append(runner.step([StepEntry(0, [token], [0])]).cpu().clone())
        manager.commit(0, 1)
    model.rt.ops.check_device_errors()
    return torch.cat(rows), model


@pytest.mark.gpu
@pytest.mark.parametrize("name, cut", [("a", 90), ("a", 3), ("b", 150), ("b", 40)])
def test_logits_over_rounded_weights(name, cut, model_folders):
    """
    The plain implementation rounds to bfloat16 where the engine does, but for gate and up, which the engine's activation reads unrounded
    here (two roundings of 2^-9 fewer): the bound of the bfloat16 replay holds, 1.2 % of the largest logit.
    """
    ids = ru.random_ids(RAW[name]["vocab_size"], cut + 20, 5)
    cfg, tensors = rounded_tensors(model_folders[name])
    want = plain.logits(cfg, tensors, ids, "bfloat16")
    got, model = engine_logits(model_folders[name], PAGES[name], ids, cut, {"weight_format": "mxfp4"})
    torch.testing.assert_close(got.double(), want, atol=0.012 * want.abs().max().item(), rtol=0.0)
    assert model.rt.ops.calls.get("ts_gemm_mxfp4", 0) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("formats", [{"weight_format": "mxfp4"}, {"weight_format": "mxfp4", "activation_format": "mxfp4"}], ids=["w", "wa"])
def test_replayed_steps_give_what_steps_without_graphs_give(formats, model_folders):
    ids = ru.random_ids(TINY_B["vocab_size"], 90, 6)
    with_graphs, _ = engine_logits(model_folders["b"], PAGE_B, ids, 60, formats)
    without, _ = engine_logits(model_folders["b"], PAGE_B, ids, 60, formats, graphs=False)
    assert torch.equal(with_graphs, without) and bool(torch.isfinite(without).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_feed_forward_is_its_operators_one_behind_the_other(rows):
    """Both formats: what the part computes is quantisation, gated product, quantisation, product, bit for bit."""
    from tinyserve_llm_b200.config.spec import GatedMLPSpec, PlainMLPSpec
    from tinyserve_llm_b200.ops import get_ops
    from tinyserve_llm_b200.parts.base import Runtime, part_class
    from tinyserve_llm_b200.parts import mlp  # noqa: F401
    ops, gen = get_ops(), torch.Generator().manual_seed(3)
    draw = lambda *shape: (0.05 * torch.randn(shape, generator=gen)).to(torch.bfloat16).cuda()  # noqa: E731
    tensors = {"gate": draw(200, 128), "up": draw(200, 128), "down": draw(128, 200)}
    x = draw(rows, 128) * 20
    up, down = ops.quantize_mxfp4(torch.cat([tensors["gate"], tensors["up"]])), ops.quantize_mxfp4(tensors["down"])
    for activation_format in (None, "mxfp4"):
        rt = Runtime(torch.bfloat16, torch.device("cuda"), ops, weight_format="mxfp4", activation_format=activation_format)
        q = ops.quantize_mxfp4 if activation_format else (lambda t: t)
        spec = GatedMLPSpec(hidden_size=128, intermediate_size=200, activation="silu", tensor_names=("gate", "up", "down"))
        got = part_class("feed_forward", spec)(spec, tensors, rt).forward(x, None)
        assert torch.equal(got, ops.linear_mxfp4(q(ops.linear_gated_mxfp4(q(x), up, "silu")), down))
        spec = PlainMLPSpec(hidden_size=128, intermediate_size=200, activation="relu2", tensor_names=("up", "down"))
        got = part_class("feed_forward", spec)(spec, tensors, rt).forward(x, None)
        h = ops.unary_activation(ops.linear_mxfp4(q(x), ops.quantize_mxfp4(tensors["up"])), "relu2")
        assert torch.equal(got, ops.linear_mxfp4(q(h), down))
        assert rt.shared["quantized_bytes"] > 0


@pytest.mark.gpu
def test_a_model_without_such_parts_is_refused(tmp_path):
    from tinyserve_llm_b200.engine import loading
    from tinyserve_llm_b200.parts.linear import QuantizedLinear
    from tinyserve_llm_b200.parts.base import Runtime
    from tinyserve_llm_b200.ops import get_ops
    rt = Runtime(torch.bfloat16, torch.device("cuda"), get_ops(), weight_format="mxfp4")
    with pytest.raises(NotImplementedError, match="multiples of 8"):
        QuantizedLinear(torch.zeros((8, 60), device="cuda"), rt)
    with pytest.raises(ValueError, match="dtype bfloat16"):
        loading.load_model(str(tmp_path), "float32", "cuda", weight_format="mxfp4")


@pytest.mark.gpu
def test_trace_replay_takes_the_formats(model_folders, tmp_path):
    proc = subprocess.run(
        [sys.executable, ru.TRACE_RUN, "--model", model_folders["a"], "--dtype", "bfloat16", "--out", str(tmp_path), "--max-tokens", "128",
         "--weight-format", "mxfp4", "--activation-format", "mxfp4"],
        input=json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [2]}], "end": ["a"]}) + "\n",
        capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0 and proc.stdout.split() == ["done", "0"], proc.stderr[-3000:]
    calls = json.loads((tmp_path / "stats.json").read_text())["kernel_calls"]
    assert calls["ts_gemm_mxfp4"] == 4 * TINY_A["num_hidden_layers"] and calls["ts_quantize_mxfp4"] == 2 * calls["ts_gemm_mxfp4"]


@pytest.mark.gpu
def test_generate_and_the_command_line(model_folders, tmp_path):
    from tinyserve_llm_b200 import LLM, CacheConfig, SamplingParams, SchedulerConfig
    folder, prompts = model_folders["a"], [[1, 2, 3, 4], [9, 8, 7]]
    llm = LLM(folder, SchedulerConfig(max_model_len=200, max_num_seqs=4, max_num_batched_tokens=256, eos_token_id=-2),
              CacheConfig(block_size=PAGE_A), num_blocks=32, weight_format="mxfp4")
    done = llm.generate(prompts, SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    out = tmp_path / "record.json"
    proc = subprocess.run(
        [sys.executable, "-m", "tinyserve_llm_b200.cli.generate", "--model", folder, "--prompt-ids", "1,2,3,4", "--prompt-ids", "9,8,7",
         "--max-tokens", "6", "--temperature", "0", "--ignore-eos", "--num-blocks", "32", "--block-size", str(PAGE_A), "--max-model-len", "200",
         "--max-num-seqs", "4", "--max-num-batched-tokens", "256", "--weight-format", "mxfp4", "--out", str(out)],
        capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stderr[-3000:]
    record = json.loads(out.read_text())
    assert record["weight_format"] == "mxfp4" and "weights mxfp4" in proc.stdout
    assert [c["token_ids"] for c in record["completions"]] == [c.token_ids for c in done]
