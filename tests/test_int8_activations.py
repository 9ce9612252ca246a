"""Which forwards take 8-bit activations: prompts', however many rows a verify or decode step has."""

from __future__ import annotations

import warnings
from dataclasses import replace
from types import SimpleNamespace

import pytest
import torch

from nanoengine_amd import kernels, model_runner, qwen3
from nanoengine_amd.config import EngineSettings
from nanoengine_amd.memory import KVCachePool, PagedSlotAllocator
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.qwen3 import AttentionBatch, Qwen3VerifyModel, Qwen3Weights, random_state_dict
from nanoengine_amd.runtime import create_verify_engine
from nanoengine_amd.sequence_state import Sequence
from test_answers import CFG, request, unit_norms
from test_draft_gpu import DCFG
from test_draft_gpu import engine as draft_engine

CPU = torch.device("cpu")
SMALL = replace(CFG, vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=4,
                num_key_value_heads=2)


class Recorder:
    """A model that keeps the batches it is given."""

    max_rows = 1 << 20
    eager_workspace = None
    config = SimpleNamespace(num_attention_heads=16, num_key_value_heads=8)

    def __init__(self):
        self.batches = []

    def ensure_rope(self, positions):
        pass

    def forward(self, rows, tokens, batch, pool, workspace=None):
        self.batches.append(batch)
        return torch.zeros(rows, 8)

    def compute_logits(self, hidden):
        return hidden, None


def test_a_steps_batch_says_whether_its_rows_are_prompts():
    """A step of the model runner is a prompt's where no row is past its sequence's prompt: an answer's next
    tokens, a sequence's guesses and steps that mix them with prompts are not."""
    model = Recorder()
    pool = SimpleNamespace(block_size=16, scratch_slot=0, key_caches=[], value_caches=[], key_scales=None, value_scales=None)
    allocator = PagedSlotAllocator(64, 16, CPU)
    runner = ModelRunner(model, pool, allocator, CPU)
    seqs = [Sequence.from_request(request(f"{i}", list(range(20 + i)))) for i in range(3)]
    for s in seqs:
        allocator.reserve(s, 40)
    step = lambda counts=None: runner._forward(model_runner.build_step_inputs(seqs, allocator, pool, CPU, counts), seqs)
    step([7, 20, 22])  # chunks of prompts, and whole ones
    seqs[0].num_cached_tokens = 7
    for s in seqs[1:]:
        s.num_cached_tokens = s.num_tokens
        s.token_ids.append(5)
    step()  # the rest of a prompt beside answers' tokens
    seqs[0].num_cached_tokens = 20
    seqs[0].token_ids.append(5)
    step()
    assert [b.prompt for b in model.batches] == [True, False, False]
    other = Sequence.from_request(request("3", list(range(30))))
    allocator.reserve(other, 40)
    runner.score_tokens(other, 30)
    other.token_ids += [4, 5, 6]
    runner.score_tokens(other, 3)
    assert [b.prompt for b in model.batches[3:]] == [True, False]


def test_a_model_too_small_for_8_bit_activations_says_so():
    state = random_state_dict(SMALL, seed=0, std=0.02)
    weights = Qwen3Weights.from_state_dict(SMALL, state, CPU, torch.bfloat16)
    with pytest.warns(UserWarning, match="int8_activations has no effect: forwards have at most 1535 rows"):
        Qwen3VerifyModel(weights, 1535, CPU, int8_activations=True)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert Qwen3VerifyModel(weights, 1535, CPU).codes is None
        assert Qwen3VerifyModel(weights, 1536, CPU, int8_activations=True).codes is not None


@pytest.mark.gpu
def test_a_prompt_into_a_cache_without_8_bit_products_says_so(monkeypatch):
    """An int8 cache with fp32 scales, which the fused products do not take, and a model that does not fuse."""
    monkeypatch.setattr(qwen3, "W8A8_MIN_ROWS", 100)
    dev = torch.device("cuda")
    weights = Qwen3Weights.from_state_dict(SMALL, random_state_dict(SMALL, seed=0, std=0.02), dev, torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=dev)
    at, n = torch.arange(112, **i32), torch.tensor([112], **i32)
    batch = AttentionBatch(at, at, torch.tensor([0], **i32), n, n, torch.arange(7, **i32)[None], 112, 112)
    for dtype, fuse in ((torch.float32, True), (torch.bfloat16, False)):
        pool = KVCachePool(1, 2, 128, 128, dev, dtype, True, 16)
        models = [Qwen3VerifyModel(weights, 128, dev, int8_activations=int8) for int8 in (True, False)]
        for model in models:
            model.fuse_qkv = fuse
        with pytest.warns(UserWarning, match="int8_activations has no effect"):
            got = models[0].forward(112, at, batch, pool).clone()
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            assert torch.equal(got, models[1].forward(112, at, batch, pool))


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_large_verify_steps_keep_16_bit_activations(graphs, monkeypatch):
    """320 slots of five rows: a verify step has more rows than a prompt needs to take the 8-bit products, and
    runs none of them, so that short prompts' tokens are those of an engine without."""
    calls = []
    fused = kernels.w8a8_qkv_norm_rope_kv
    monkeypatch.setattr(kernels, "w8a8_qkv_norm_rope_kv", lambda codes, *a, **kw: calls.append(codes.shape[0]) or fused(codes, *a, **kw))
    tokens = []
    for int8 in (True, False):
        settings = EngineSettings(device="cuda", dtype="bfloat16", kv_cache="paged", scheduler="continuous", quantization="int8",
                                  int8_activations=int8, kv_cache_dtype="int8", speculative="ngram", num_speculative_tokens=4,
                                  ngram_max_size=3, max_num_seqs=320, max_model_len=1700, kv_cache_memory_mb=64,
                                  cuda_graphs=graphs, cuda_graph_max_batch=320, cuda_graph_max_context=1700)
        runner = create_verify_engine(CFG, unit_norms(), settings, max_prefill_rows=1600).runner
        assert runner.max_seqs * runner.R >= qwen3.W8A8_MIN_ROWS
        seqs = [Sequence.from_request(request(f"{i}", [5 + i, 6, 7, 8] * (3 + i), ignore_eos=True, seed=i)) for i in range(6)]
        runner.add(seqs)
        while min(s.num_generated_tokens for s in seqs) < 16:
            runner.step()
        while runner.pending:
            runner.step()
        tokens.append([s.token_ids[: s.num_prompt_tokens + 16] for s in seqs])
        assert calls == []
        long = Sequence.from_request(request("long", [9, 8, 7, 6] * 400, ignore_eos=True, seed=9))
        runner.add([long])
        runner.step()
        assert calls == ([1600] * CFG.num_hidden_layers if int8 else [])
        calls.clear()
    assert tokens[0] == tokens[1]


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_a_draft_models_prompts_are_told_from_its_guesses(graphs):
    """Of a draft model's forwards only those over its requests' prompts say that they are prompts'."""
    runner = draft_engine(unit_norms(), DCFG, random_state_dict(DCFG, seed=7, std=0.02), 2, graphs=graphs).runner
    model, seen = runner.proposer.model, []
    plain = model.forward
    model.forward = lambda rows, tokens, batch, *a, **kw: seen.append((rows, batch.prompt)) or plain(rows, tokens, batch, *a, **kw)
    runner.add([Sequence.from_request(request(f"{i}", [5, 6, 7, 8] * 5 + [i], ignore_eos=True)) for i in range(2)])
    for _ in range(4):
        runner.step()
    prompts = [rows for rows, prompt in seen if prompt]
    assert prompts == [44] and len(seen) > 1  # (each prompt with the target's first token)
