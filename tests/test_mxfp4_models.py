"""Models held in microscaled 4-bit floating point: layers wide enough that decode steps go in pieces, and a model with no part that takes it."""

from __future__ import annotations

import pytest
import torch

import nipizen_configs
import plain_llama as plain
import replay_util as ru
from test_mxfp4_engine import rounded_tensors
from tiny_configs import TINY_A, WEIGHTS

PAGE = 16
WIDE = dict(TINY_A, hidden_size=512, intermediate_size=5632, num_attention_heads=8, num_key_value_heads=4)


@pytest.fixture(scope="module")
def wide_folder(tmp_path_factory):
    from tinyserve_llm_b200.weights import write_random_model
    folder = str(tmp_path_factory.mktemp("wide"))
    write_random_model(folder, WIDE, 17, **WEIGHTS)
    return folder


def decode(folder, requests, cut, graphs):
    """Logits of every request's last tokens: all first `cut` tokens in one step, then step by step, every request one token."""
    from tinyserve_llm_b200.engine.loading import build_cache, load_model
    from tinyserve_llm_b200.engine.step import StepEntry, StepRunner
    model = load_model(folder, "bfloat16", "cuda", weight_format="mxfp4")
    _, manager, storage = build_cache(model, PAGE, 64, caching=False)
    runner = StepRunner(model, manager, storage, cuda_graphs=graphs)
    for i, ids in enumerate(requests):
        assert manager.admit(i, ids[:cut])
    rows = [runner.step([StepEntry(i, ids[:cut], [cut - 1]) for i, ids in enumerate(requests)]).cpu().clone()]
    for i in range(len(requests)):
        manager.commit(i, cut)
    for at in range(cut, len(requests[0])):
        for i, ids in enumerate(requests):
            manager.extend(i, [ids[at]])
        rows.append(runner.step([StepEntry(i, [ids[at]], [0]) for i, ids in enumerate(requests)]).cpu().clone())
        for i in range(len(requests)):
            manager.commit(i, 1)
    model.rt.ops.check_device_errors()
    return torch.stack(rows, dim=1), model.rt.ops


@pytest.mark.gpu
def test_decode_steps_in_pieces(wide_folder):
    """Ten requests decoding: gate and up go in pieces.  Bound as in test_mxfp4_engine.py, 1.2 % of the largest logit."""
    requests = [ru.random_ids(WIDE["vocab_size"], 12, 90 + i) for i in range(10)]
    cut = 6
    got, ops = decode(wide_folder, requests, cut, True)
    assert ops.lib.ts_gemm_mxfp4_scratch_bytes(10, 2 * WIDE["intermediate_size"], WIDE["hidden_size"], 0, 1) > 0
    without, _ = decode(wide_folder, requests, cut, False)
    assert torch.equal(got, without)
    cfg, tensors = rounded_tensors(wide_folder)
    for i, ids in enumerate(requests):
        want = plain.logits(cfg, tensors, ids, "bfloat16")[cut - 1:]
        torch.testing.assert_close(got[i].double(), want, atol=0.012 * want.abs().max().item(), rtol=0.0)


@pytest.mark.gpu
def test_a_model_that_holds_nothing_in_four_bits_is_refused(tmp_path):
    """Gated attention, delta rules and routed experts alone: no projection of the model takes the format."""
    from tinyserve_llm_b200.engine.loading import load_model
    from tinyserve_llm_b200.weights import write_random_model
    write_random_model(str(tmp_path), nipizen_configs.MIXED, 3, **nipizen_configs.WEIGHTS)
    with pytest.raises(ValueError, match="no part of this model"):
        load_model(str(tmp_path), "bfloat16", "cuda", weight_format="mxfp4")
    assert load_model(str(tmp_path), "bfloat16", "cuda").rt.weight_format is None
