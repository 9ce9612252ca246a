"""Requests with penalties, biases and allowed tokens through the model runner and the verify
runner, prompts through the 8-bit products, and a step from hidden rows to tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nanoengine_amd import kernels, qwen3
from nanoengine_amd._native import EPILOGUE_SWIGLU
from nanoengine_amd.config import EngineSettings
from nanoengine_amd.int8_quantization import Int8Linear, quantize_linear_layers
from nanoengine_amd.interface import SamplingParams, sampling_uniform
from nanoengine_amd.memory import KVCachePool
from nanoengine_amd.qwen3 import AttentionBatch, Qwen3VerifyModel, Qwen3Weights, random_state_dict
from nanoengine_amd.runtime import create_verify_engine
from nanoengine_amd.sequence_state import Sequence
from test_adjust_logits_gpu import check, reference
from test_answers import CFG, build, engine, request, unit_norms
from test_draft_gpu import DCFG
from test_draft_gpu import engine as draft_engine
from test_sample_gpu import reference_row
from test_w8a8_gpu import check_product, rows_reference


def test_parameters_and_settings():
    plain = SamplingParams(4, temperature=1.0, top_k=3)
    assert not plain.is_penalized and not plain.is_adjusted
    for kw in (dict(repetition_penalty=1.1), dict(presence_penalty=-0.5), dict(frequency_penalty=0.5)):
        assert SamplingParams(4, **kw).is_penalized and SamplingParams(4, **kw).is_adjusted
    biased = SamplingParams(4, logit_bias={3: 1.0})
    assert biased.is_adjusted and not biased.is_penalized and not SamplingParams(4, logit_bias={}).is_adjusted
    assert hash(biased) == hash(SamplingParams(4)) and biased != SamplingParams(4)
    with pytest.raises(ValueError, match="quantization"):
        EngineSettings(int8_activations=True)
    env = {"NANOENGINE_QUANTIZATION": "int8", "NANOENGINE_INT8_ACTIVATIONS": "1"}
    assert EngineSettings.from_env(env).int8_activations and not EngineSettings().int8_activations


def test_layers_keep_how_they_take_activations():
    linear = torch.nn.Linear(64, 32, bias=False)
    assert not Int8Linear.from_linear(linear).int8_activations and Int8Linear.from_linear(linear, True).int8_activations
    layer = torch.nn.Module()
    layer.self_attn, layer.mlp = torch.nn.Module(), torch.nn.Module()
    layer.mlp.down_proj = linear
    model = torch.nn.Module()
    model.model = torch.nn.Module()
    model.model.layers = [layer]
    assert quantize_linear_layers(model, int8_activations=True) == 1 and layer.mlp.down_proj.int8_activations


# ------------------------------------------------------------------ the model runner
@pytest.mark.gpu
def test_steps_with_penalties_biases_and_masks():
    """Every step's tokens are those of the 64-bit draw from the 64-bit adjusted logits of that step."""
    runner = build(unit_norms(), True, False, False, 64)
    seen = []
    compute = runner._model.compute_logits
    runner._model.compute_logits = lambda hidden, **kw: seen.append(compute(hidden, **kw)) or seen[-1]
    ways = [dict(repetition_penalty=1.3), dict(presence_penalty=0.7, frequency_penalty=0.4, temperature=0.9, seed=5),
            dict(logit_bias={7: 30.0, 4095: -5.0}), dict(temperature=0.8, top_k=20, seed=6), dict(),
            dict(temperature=1.1, top_k=50, min_p=0.01, seed=7, frequency_penalty=0.3, logit_bias={11: 2.0}), dict(temperature=0.7, seed=8)]
    g = torch.Generator().manual_seed(1)
    seqs = [Sequence.from_request(request(f"{i}", torch.randint(0, 30, (9 + i,), generator=g).tolist(), **w))
            for i, w in enumerate(ways)]
    for step in range(5):
        masks = [None] * len(seqs)
        if step >= 2:  # a greedy request and a sampled one under a grammar
            masks[4], masks[6] = [100 + step, 2000], list(range(step, 4096, 7))
        for s in seqs:
            runner.allocator.reserve(s, s.num_tokens)
        tokens = runner.run_step(seqs, allowed_tokens=None if step < 2 else masks)
        logits = seen[-1][0]
        for i, s in enumerate(seqs):
            p = s.sampling_params
            one = lambda *v: torch.tensor(v, dtype=torch.int32)
            penalties = kernels.TokenPenalties(one(s.token_ids), one(s.num_tokens), one(s.num_prompt_tokens), p.repetition_penalty,
                                               p.presence_penalty, p.frequency_penalty)
            bias = kernels.TokenBias.from_dicts([p.logit_bias], torch.device("cpu"))
            mask = kernels.allowed_mask([masks[i]], 4096, torch.device("cpu"))
            x, _ = reference(logits[i : i + 1].cpu(), penalties, bias, mask)
            if p.is_adjusted or p.is_filtered or masks[i] is not None:
                u = np.float32(sampling_uniform(s.sampling_generator.seed, step))
                want = reference_row(x[0], float(u), float(np.float32(p.temperature)), min(p.top_k, 4096),
                                     float(np.float32(p.top_p)), float(np.float32(p.min_p)))[0]
                assert tokens[i] == want
            elif p.temperature == 0:
                assert tokens[i] == int(logits[i].float().argmax())
            s.token_ids.append(tokens[i])
    assert seqs[2].token_ids[-1] == 7 and seqs[4].token_ids[-1] in (104, 2000)


@pytest.mark.gpu
def test_a_step_without_any_allowed_token_moves_nothing():
    runner = build(unit_norms(), True, False, False, 64)
    seqs = [Sequence.from_request(request(f"{i}", [1, 2, 3], temperature=1.0, seed=i)) for i in range(2)]
    for s in seqs:
        runner.allocator.reserve(s, 4)
    with pytest.raises(ValueError, match="1: no token is allowed"):
        runner.run_step(seqs, allowed_tokens=[None, []])
    assert all(s.num_cached_tokens == 0 and s.sampling_generator.step == 0 for s in seqs)
    with pytest.raises(ValueError, match="allowed_tokens for 1 of 2"):
        runner.run_step(seqs, allowed_tokens=[None])
    with pytest.raises(ValueError, match="repetition_penalty"):
        runner.run_step([Sequence.from_request(request("z", [1], repetition_penalty=0.0))])
    assert len(runner.run_step(seqs, allowed_tokens=[[5], None])) == 2 and seqs[0].num_cached_tokens == 3


# ----------------------------------------------------------------- the verify runner
def penalized(i: int, **kw) -> dict:
    return dict(seed=i, ignore_eos=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_verify_rows_count_the_guesses_before_them(temperature, monkeypatch):
    """Every row's logits under its sequence's own tokens and the guesses before it; greedy requests
    emit what those logits say."""
    runner = engine(unit_norms(), 3, False, False).runner
    runner.trace = []
    calls = []
    adjust = kernels.adjust_logits

    def spy(logits, penalties=None, **kw):
        calls.append((logits.clone(), [t.clone() for t in (penalties.history, penalties.history_len, penalties.prompt_len)]))
        out = adjust(logits, penalties, **kw)
        calls[-1] += (out.clone(),)
        return out

    monkeypatch.setattr(kernels, "adjust_logits", spy)
    params = [dict(repetition_penalty=1.2, presence_penalty=0.3), dict(), dict(frequency_penalty=0.6, temperature=temperature)]
    prompts = [[3, 4, 5, 6] * 6, [9, 8] * 10, [1, 2, 3] * 7 + [1]]
    seqs = [Sequence.from_request(request(f"{i}", prompts[i], **penalized(i, **p))) for i, p in enumerate(params)]
    runner.add(seqs)
    logits, (history, length, prompt), out = calls[0]
    first = kernels.TokenPenalties(history.cpu(), length.cpu(), prompt.cpu(), torch.tensor([1.2, 1.0, 1.0]),
                                   torch.tensor([0.3, 0.0, 0.0]), torch.tensor([0.0, 0.0, 0.6]))
    check(out, logits, penalties=first)
    assert length.tolist() == [24, 20, 22] and prompt[0] == 24 and prompt[2] == 22
    guessed = 0
    for _ in range(8):
        before = [list(s.token_ids) for s in seqs]
        calls.clear()
        runner.step()
        (logits, _, out), step = calls[0], runner.trace[-1]
        for slot, s in enumerate(seqs):
            p, drafts, r0 = s.sampling_params, step[slot]["drafts"], slot * runner.R
            assert step[slot]["history"] == before[slot]
            guessed += len(drafts)
            target = []
            for i in range(len(drafts) + 1):
                tokens = torch.tensor([before[slot] + drafts[:i]], dtype=torch.int32)
                row = kernels.TokenPenalties(tokens, torch.tensor([tokens.shape[1]]), torch.tensor([s.num_prompt_tokens]),
                                             p.repetition_penalty, p.presence_penalty, p.frequency_penalty)
                check(out[r0 + i : r0 + i + 1], logits[r0 + i : r0 + i + 1], penalties=row)
                target.append(int(out[r0 + i].float().argmax()))
            if p.temperature == 0:
                kept = 0
                while kept < len(drafts) and drafts[kept] == target[kept]:
                    kept += 1
                assert step[slot]["out"] == drafts[:kept] + [target[kept]]
                assert s.token_ids == before[slot] + drafts[:kept] + [target[kept]]
    assert guessed > 0  # (rows with guesses were among them)


@pytest.mark.gpu
def test_penalties_come_and_go_in_eager_and_captured_steps():
    state = unit_norms()
    runners = [engine(state, 4, False, graphs).runner for graphs in (False, True)]
    tokens = [[], []]
    for runner, kept in zip(runners, tokens):
        for turn in range(3):
            seqs = []
            for i in range(4):
                # (so large a presence penalty that no token comes twice)
                params = dict(presence_penalty=1000.0) if (turn, i) in ((0, 1), (1, 0), (1, 3)) else {}
                params["temperature"] = 0.9 if (turn, i) == (1, 3) else 0.0
                seqs.append(Sequence.from_request(request(f"{turn}.{i}", [5 + turn, 6, 7, 8] * 5 + [i], **penalized(i, **params))))
            runner.add(seqs)
            assert runner.any_adjusted == (turn < 2)
            while min(s.num_generated_tokens for s in seqs) < 24:
                runner.step()
            for s in seqs:
                made = s.token_ids[s.num_prompt_tokens :]
                if s.sampling_params.is_penalized:
                    assert len(set(made)) == len(made)
                kept.append(list(s.token_ids))
            for slot in runner.active_slots:
                runner.release(slot)
            while runner.pending:
                runner.step()
            assert not runner.any_adjusted and not runner.np_adjusted.any()
            assert (runner.penalties.presence == 0).all() and (runner.penalties.repetition == 1).all()
    for a, b in zip(*tokens):
        n = min(len(a), len(b))
        assert a[:n] == b[:n]
    assert runners[1].graph is not None and runners[1].graph_adjusted is False


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_penalties_with_a_draft_models_guesses(graphs):
    """The target's penalties hold whatever another model guesses, greedy and sampled: no token comes
    twice under so large a penalty."""
    draft = random_state_dict(DCFG, seed=7, std=0.02)
    ways = [dict(presence_penalty=1000.0), dict(presence_penalty=1000.0, temperature=0.8), dict(),
            dict(frequency_penalty=1000.0, temperature=1.2)]
    runner = draft_engine(unit_norms(), DCFG, draft, len(ways), graphs=graphs).runner
    runner.trace = None if graphs else []
    seqs = [Sequence.from_request(request(f"{i}", [5, 6, 7, 8] * 5 + [i], **penalized(i, **w))) for i, w in enumerate(ways)]
    runner.add(seqs)
    while min(s.num_generated_tokens for s in seqs) < 24:
        runner.step()
    assert runner.proposer.forwards > 0 and runner.any_adjusted
    assert not graphs or (runner.graph is not None and runner.graph_adjusted)
    for s, way in zip(seqs, ways):
        made = s.token_ids[s.num_prompt_tokens :]
        assert len(set(made)) == len(made) or not way
    for step in runner.trace or []:  # what was kept was guessed
        for rec in step.values():
            kept = len(rec["out"]) - 1
            assert rec["out"][:kept] == rec["drafts"][:kept]


@pytest.mark.gpu
def test_verification_refuses_what_it_does_not_take():
    runner = engine(unit_norms(), 2, False, False).runner
    for kw in (dict(logit_bias={1: 1.0}), dict(repetition_penalty=0.0), dict(repetition_penalty=float("inf"))):
        with pytest.raises(ValueError):
            runner.add([Sequence.from_request(request("a", [1, 2], **kw))])
    assert runner.free_slots() == [0, 1]


# ---------------------------------------------------------------- prompts in 8 bits
@pytest.mark.gpu
@pytest.mark.parametrize("int8_cache", [True, False])
def test_prompts_through_the_8_bit_products(int8_cache, monkeypatch):
    """The model's forward against the same calls made one by one, bit for bit, and near the forward
    with 16-bit activations: a row's codes are off by at most half of its largest value / 127, at most
    max/rms / (127 sqrt 12) of its rms each time (max/rms < 8 here), and four such products a layer over
    two layers add up to at most sqrt(8) of that: 5.2e-2."""
    monkeypatch.setattr(qwen3, "W8A8_MIN_ROWS", 100)
    dev = torch.device("cuda")
    weights = Qwen3Weights.from_state_dict(CFG, unit_norms(), dev, torch.bfloat16)
    rows = 150
    model, other = Qwen3VerifyModel(weights, 160, dev, int8_activations=True), Qwen3VerifyModel(weights, 160, dev)
    pools = [KVCachePool(2, 8, 128, 512, dev, torch.bfloat16, int8_cache, 16) for _ in range(3)]
    i32 = dict(dtype=torch.int32, device=dev)
    tokens = torch.randint(0, 4096, (rows,), generator=torch.Generator().manual_seed(0)).to(**i32)
    positions = torch.cat([torch.arange(90, **i32), torch.arange(60, **i32)])
    slots = torch.cat([torch.arange(90, **i32), torch.arange(96, 156, **i32)])
    tables = torch.stack([torch.arange(6, **i32), torch.arange(6, 12, **i32)])
    lengths = torch.tensor([90, 60], **i32)
    batch = AttentionBatch(positions, slots, torch.tensor([0, 90], **i32), lengths, lengths, tables, 90, 90)
    got = model.forward(rows, tokens, batch, pools[0]).clone()
    near = other.forward(rows, tokens, batch, pools[1]).clone()
    assert float((got.float() - near.float()).norm() / near.float().norm()) < 5.2e-2
    assert not torch.equal(got, near)

    pool, c, eps = pools[2], CFG, CFG.rms_norm_eps
    res, x = kernels.embed_rmsnorm(tokens, weights.embed, weights.layers[0].input_layernorm, eps)
    for i, layer in enumerate(weights.layers):
        qkv = kernels.w8a8_gemm(*kernels.quantize_rows(x), layer.qkv_int8, layer.qkv_scale)
        q = kernels.qk_norm_rope_kv_write(qkv, c.num_attention_heads, c.num_key_value_heads, layer.q_norm, layer.k_norm, eps,
                                          positions, model.rope, slots, pool.key_caches[i], pool.value_caches[i],
                                          pool.key_scale_2d(i), pool.value_scale_2d(i))
        attn = kernels.paged_verify_attention(q, pool.key_caches[i], pool.value_caches[i], pool.key_scale_2d(i),
                                              pool.value_scale_2d(i), tables, 16, lengths, batch.q_start, lengths, 90, 90)
        delta = kernels.w8a8_gemm(*kernels.quantize_rows(attn.view(rows, -1)), layer.o_int8, layer.o_scale)
        x = kernels.add_rmsnorm(res, delta, layer.post_attention_layernorm, eps)
        act = kernels.w8a8_gemm(*kernels.quantize_rows(x), layer.gate_up_int8, layer.gate_up_scale, epilogue=EPILOGUE_SWIGLU)
        delta = kernels.w8a8_gemm(*kernels.quantize_rows(act), layer.down_int8, layer.down_scale)
        x = kernels.add_rmsnorm(res, delta, weights.layers[i + 1].input_layernorm if i == 0 else weights.norm, eps)
    assert torch.equal(got, x)
    # fewer rows keep 16-bit activations
    few = AttentionBatch(positions[:90], slots[:90], batch.q_start[:1], lengths[:1], lengths[:1], tables[:1], 90, 90)
    assert torch.equal(model.forward(90, tokens, few, pools[0]), other.forward(90, tokens, few, pools[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["int8", "auto"])
def test_an_engines_prompts_in_8_bits_and_its_steps_in_16(cache, monkeypatch):
    """Prompts of many rows take the 8-bit products, short ones and verify steps do not, captured or not."""
    monkeypatch.setattr(qwen3, "W8A8_MIN_ROWS", 100)
    rows = []
    fused = kernels.w8a8_qkv_norm_rope_kv
    monkeypatch.setattr(kernels, "w8a8_qkv_norm_rope_kv", lambda codes, *a, **kw: rows.append(codes.shape[0]) or fused(codes, *a, **kw))
    tokens = []
    for graphs in (False, True):
        settings = EngineSettings(device="cuda", dtype="bfloat16", kv_cache="paged", scheduler="continuous", quantization="int8",
                                  int8_activations=True, kv_cache_dtype=cache, speculative="ngram", num_speculative_tokens=4,
                                  ngram_max_size=3, max_num_seqs=4, max_model_len=400, kv_cache_memory_mb=64, cuda_graphs=graphs,
                                  cuda_graph_max_batch=4, cuda_graph_max_context=400)
        runner = create_verify_engine(CFG, unit_norms(), settings, max_prefill_rows=160).runner
        seqs = [Sequence.from_request(request(f"{i}", [5 + i, 6, 7, 8] * n, ignore_eos=True, seed=i, presence_penalty=0.1 * i))
                for i, n in enumerate((14, 9, 16))]
        runner.add(seqs)
        late = Sequence.from_request(request("3", [1, 2, 3], ignore_eos=True))
        runner.add([late])
        while late.num_generated_tokens < 12:
            runner.step()
        while runner.pending:
            runner.step()
        tokens.append([s.token_ids[: s.num_prompt_tokens + 12] for s in (*seqs, late)])
    assert rows == [156] * CFG.num_hidden_layers * 2 and tokens[0] == tokens[1]


@pytest.mark.gpu
def test_layer_with_8_bit_activations():
    linear = torch.nn.Linear(272, 100, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = Int8Linear.from_linear(linear, int8_activations=True)
    x = torch.randn(3, 5, 272, device="cuda").bfloat16()
    codes, scales = rows_reference(x.view(15, 272))
    y = layer(x)
    assert y.shape == (3, 5, 100)
    check_product(y.view(15, 100), codes, scales, layer.weight_int8, layer.weight_scale)
    check_product(layer(x[:, 0])[:, :], *rows_reference(x[:, 0].contiguous()), layer.weight_int8, layer.weight_scale)


# --------------------------------------------------------- from hidden rows to tokens
@pytest.mark.gpu
def test_step_from_hidden_rows_to_tokens():
    """Norm, 8-bit output head, adjustment and draw as one captured step, replayed as histories grow,
    against the draw from the 64-bit product of the same codes."""
    b, hidden, vocab, steps = 6, 256, 5003, 4
    g = torch.Generator(device="cuda").manual_seed(4)
    head = torch.nn.Linear(hidden, vocab, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = Int8Linear.from_linear(head)
    weight = torch.rand(hidden, device="cuda", generator=g).bfloat16()
    x = torch.empty(b, hidden, device="cuda", dtype=torch.bfloat16)
    u = torch.empty(b, device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    history, length = torch.zeros(b, 64, **i32), torch.full((b,), 3, **i32)
    penalties = kernels.TokenPenalties(history, length, torch.full((b,), 2, **i32), 1.5, 0.25, 0.5)
    mask = kernels.allowed_mask([None, list(range(0, vocab, 3)), [4, 5002], None, list(range(100)), None], vocab, x.device)
    logits = torch.empty(b, vocab, device="cuda", dtype=torch.bfloat16)
    adjusted = torch.empty(b, vocab, device="cuda")
    codes, scales = torch.empty(b, hidden, device="cuda", dtype=torch.int8), torch.empty(b, device="cuda")
    tokens = torch.empty(b, **i32)

    def step():
        kernels.rmsnorm_quantize(x, weight, 1e-6, codes=codes, scales=scales)
        kernels.w8a8_gemm(codes, scales, layer.weight_int8, layer.weight_scale, out=logits)
        kernels.adjust_logits(logits, penalties, allowed=mask, out=adjusted)
        kernels.sample(adjusted, u, temperature=0.7, top_k=40, out=tokens)

    x.normal_()
    u.fill_(0.5)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for s in range(steps):
        x.copy_(torch.randn(b, hidden, device="cuda", generator=g))
        u.copy_(torch.rand(b, device="cuda", generator=g))
        graph.replay()
        drawn = tokens.tolist()
        torch.cuda.synchronize()
        check_product(logits, codes, scales, layer.weight_int8, layer.weight_scale)
        check(adjusted, logits, penalties=penalties, allowed=mask)
        for r in range(b):
            assert drawn[r] == reference_row(adjusted[r].double().cpu().numpy(), float(u[r]), float(np.float32(0.7)), 40, 1.0, 0.0)[0]
        replayed = tokens.clone()
        step()
        assert torch.equal(tokens, replayed)
        history[torch.arange(b), length.long()] = tokens
        length += 1
