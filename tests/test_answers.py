"""Many answers to one prompt: a prompt's sequence forked for each of them, their shared blocks
read once a step, their tokens drawn under filters of their own -- through the model runner and
the verify runner."""

from __future__ import annotations

import random
from dataclasses import replace

import numpy as np
import pytest
import torch

from nanoengine_amd import kernels
from nanoengine_amd.config import EngineSettings
from nanoengine_amd.interface import GenerationRequest, SamplingParams, sampling_uniform
from nanoengine_amd.memory import KVCachePool, PagedSlotAllocator, PrefixCachingSlotAllocator, find_shared_prefixes
from nanoengine_amd.model_runner import ModelRunner
from nanoengine_amd.qwen3 import QWEN3_0_6B, Qwen3VerifyModel, Qwen3Weights, random_state_dict
from nanoengine_amd.runtime import create_verify_engine
from nanoengine_amd.sequence_state import Sequence
from oracle import accept as oracle_accept
from test_sample_gpu import reference_row

CFG = replace(QWEN3_0_6B, vocab_size=4096, num_hidden_layers=2)
CPU = torch.device("cpu")


def request(rid: str, tokens: list[int], **params) -> GenerationRequest:
    return GenerationRequest(rid, tokens, SamplingParams(max_new_tokens=64, **params))


# ------------------------------------------------------------------------- host
def best_saving(tables: list[tuple]) -> int:
    """The most that groups can save, tried out over the tree of first blocks."""
    def solve(members: list[tuple], depth: int) -> int:
        if len(members) < 2:
            return 0
        heads: dict = {}
        for t in members:
            heads.setdefault(t[depth] if len(t) > depth else ("end", id(t)), []).append(t)
        inner = sum(solve(m, depth + 1) for key, m in heads.items() if not isinstance(key, tuple))
        return max(inner, (len(members) - 1) * depth)
    return solve(tables, 0)


@pytest.mark.parametrize("seed", range(40))
def test_shared_prefixes_save_the_most(seed):
    r = random.Random(seed)
    tables = [[r.randrange(2) for _ in range(r.randrange(9))] for _ in range(r.randrange(1, 14))]
    # a block belongs to one prefix: name it by its path
    tables = [[int("1" + "".join(map(str, t[: i + 1])), 3) for i in range(len(t))] for t in tables]
    found = find_shared_prefixes(tables)
    members = [i for group, _ in found for i in group]
    assert len(members) == len(set(members)) and all(len(g) > 1 and n > 0 for g, n in found)
    for group, n in found:
        assert len({tuple(tables[i][:n]) for i in group}) == 1 and min(len(tables[i]) for i in group) >= n
    assert sum((len(g) - 1) * n for g, n in found) == best_saving([tuple(t) for t in tables])


def test_shared_prefixes_of_many_tables():
    assert find_shared_prefixes([]) == [] and find_shared_prefixes([[], [3], []]) == []
    chain = [list(range(i + 1)) for i in range(1100)]  # each one block longer than the one before
    (group, blocks), = [f for f in find_shared_prefixes(chain) if len(f[0]) > 2]
    assert group == list(range(blocks - 1, 1100)) and (1100 - blocks) * blocks == 550 * 550
    same = [np.arange(5) for _ in range(64)]
    assert find_shared_prefixes(same) == [(list(range(64)), 5)]
    assert find_shared_prefixes([[7, 8, 1], [9, 2], [7, 8, 3], [9, 4], [5]]) == [([0, 2], 2), ([1, 3], 1)]


@pytest.mark.parametrize("seed,step", [(0, 0), (1, 7), (2**62 + 12345, 3), (99, 2**33 + 5), (2**40, 2**31)])
def test_a_streams_uniform_is_the_acceptance_kernels_draw(seed, step):
    assert sampling_uniform(seed, step) == oracle_accept.uniform(seed, step, 63)


def test_settings_and_parameters():
    with pytest.raises(ValueError, match="prefix_cache"):
        EngineSettings(kv_cache="paged", shared_prefix=True)
    env = {"NANOENGINE_KV_CACHE": "paged", "NANOENGINE_PREFIX_CACHE": "1", "NANOENGINE_SHARED_PREFIX": "true"}
    assert EngineSettings.from_env(env).shared_prefix and not EngineSettings().shared_prefix
    assert not SamplingParams(4).is_filtered and not SamplingParams(4, temperature=1.0, top_p=0.5).is_filtered
    assert not SamplingParams(4, top_k=5, min_p=0.1).is_filtered  # greedy
    assert SamplingParams(4, temperature=1.0, top_k=5).is_filtered
    assert SamplingParams(4, temperature=1.0, min_p=0.1).is_filtered


class Copies:
    block_size = 16

    def __init__(self):
        self.pairs = []

    def copy_blocks(self, src, dst):
        self.pairs.append((src, dst))


@pytest.mark.parametrize("caching", [False, True])
def test_fork_starts_from_the_cached_tokens(caching):
    pool = Copies()
    allocator = (PrefixCachingSlotAllocator if caching else PagedSlotAllocator)(16, 16, CPU)
    runner = ModelRunner(None, pool, allocator, CPU)
    parent = Sequence.from_request(request("p", list(range(40))))
    allocator.reserve(parent, 40)
    parent.num_cached_tokens = 40
    same = runner.fork(parent, request("same", list(range(40))))  # its last token is left to compute
    longer = runner.fork(parent, request("longer", list(range(40)) + [7, 8]))
    assert same.num_cached_tokens == 39 and longer.num_cached_tokens == 40
    assert [len(src) for src, _ in pool.pairs] == ([1, 1] if caching else [3, 3])
    assert (allocator.block_table(same)[:2] == allocator.block_table(parent)[:2]) == caching
    with pytest.raises(ValueError, match="does not start with"):
        runner.fork(parent, request("other", [9] + list(range(1, 41))))
    with pytest.raises(ValueError, match="already holds"):
        runner.fork(parent, request("same", list(range(40))))
    assert len(pool.pairs) == 2 and runner.fork(parent, request("one", [0])).num_cached_tokens == 0


# -------------------------------------------------------------------------- GPU
def unit_norms() -> dict:
    state = random_state_dict(CFG, seed=0, std=0.02)
    return {n: torch.ones_like(t) if n.endswith("norm.weight") or "layernorm" in n else t for n, t in state.items()}


def build(state, int8: bool, caching: bool, shared: bool, blocks: int) -> ModelRunner:
    dev = torch.device("cuda")
    model = Qwen3VerifyModel(Qwen3Weights.from_state_dict(CFG, state, dev, torch.bfloat16), 160, dev)
    pool = KVCachePool(2, 8, 128, blocks * 16, dev, torch.bfloat16, int8, 16)
    allocator = (PrefixCachingSlotAllocator if caching else PagedSlotAllocator)(blocks, 16, dev)
    return ModelRunner(model, pool, allocator, dev, shared_prefix=shared)


def rel(got, ref) -> float:
    return float((got.float() - ref.float()).norm() / ref.float().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("int8,members", [(True, 70), (False, 36)])
def test_answers_of_a_forked_prompt(int8, members, monkeypatch):
    """A prompt computed once and forked ``members`` times, three steps each, against the same
    with copied blocks and ordinary attention: logits as near as two bf16 forwards are, tokens
    those of the 64-bit draw from the logits of the step."""
    state = unit_norms()
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, 4096, (1557,), generator=g).tolist()
    ways = [dict(temperature=0.8, top_k=20), dict(temperature=1.3, min_p=0.05, top_p=0.9), dict(temperature=0.6),
            dict(), dict(temperature=1.0, top_k=1 + 4096, min_p=0.01)]
    plans, logits = [], []
    plan = kernels.shared_prefix_plan
    monkeypatch.setattr(kernels, "shared_prefix_plan", lambda *a, **k: plans.append(plan(*a, **k)) or plans[-1])

    def start(shared: bool):
        runner = build(state, int8, shared, shared, 110 + members * (8 if shared else 104))
        compute = runner._model.compute_logits

        def spy(hidden, **kw):
            out = compute(hidden, **kw)
            logits.append(out[0])
            return out
        runner._model.compute_logits = spy
        parent = Sequence.from_request(request("parent", prompt))
        runner.allocator.reserve(parent, parent.num_tokens)
        while parent.num_uncached_tokens:
            runner.run_step([parent], [min(150, parent.num_uncached_tokens)])
        seqs = []
        for i in range(members):
            params = dict(seed=100 + i, **ways[i % len(ways)])
            seqs.append(runner.fork(parent, request(f"r{i}", prompt + ([i] if i % 3 else []), **params)))
        return runner, seqs

    ours, seqs = start(True)
    other, theirs = start(False)
    assert not plans
    for step in range(3):
        logits.clear()
        for runner, batch in ((ours, seqs), (other, theirs)):
            for s in batch:
                runner.allocator.reserve(s, s.num_tokens)
        tokens, before = ours.run_step(seqs), len(plans)
        other.run_step(theirs)
        assert len(plans) == before == step + 1 and plans[-1].error_flag() == 0 and plans[-1].shared_items() > 0
        assert rel(logits[0], logits[1]) <= 2e-2
        x = logits[0].double().cpu().numpy()
        for i, s in enumerate(seqs):
            p = s.sampling_params
            if p.is_filtered or p.temperature == 0.0:
                u = np.float32(sampling_uniform(s.sampling_generator.seed, step))
                want = reference_row(x[i], float(u), float(np.float32(p.temperature)), min(p.top_k, 4096),
                                     float(np.float32(p.top_p)), float(np.float32(p.min_p)))[0]
                assert tokens[i] == want
            assert s.sampling_generator.step == (step + 1 if p.temperature else 0)
            assert s.num_cached_tokens == s.num_tokens == theirs[i].num_cached_tokens
            s.token_ids.append(tokens[i])
            theirs[i].token_ids.append(tokens[i])
    only = [s for s in seqs if s.sampling_params.is_filtered]
    for s in only:
        ours.allocator.reserve(s, s.num_tokens)
    logits.clear()
    tokens = ours.run_step(only)
    for i, s in enumerate(only):
        p = s.sampling_params
        want = reference_row(logits[0][i].double().cpu().numpy(), float(np.float32(sampling_uniform(s.sampling_generator.seed, 3))),
                             float(np.float32(p.temperature)), min(p.top_k, 4096), float(np.float32(p.top_p)),
                             float(np.float32(p.min_p)))[0]
        assert tokens[i] == want and s.sampling_generator.step == 4
        s.token_ids.append(tokens[i])
    ours.allocator.reserve(seqs[0], seqs[0].num_tokens)
    made = len(plans)
    for s in seqs[1:]:
        ours.allocator.free(s)
    few = ours.run_step([seqs[0]])  # one answer left: nothing is shared, nothing is planned
    assert len(plans) == made and len(few) == 1


def engine(state, members: int, shared: bool, graphs: bool):
    settings = EngineSettings(device="cuda", dtype="bfloat16", kv_cache="paged", scheduler="continuous",
                              quantization="int8", kv_cache_dtype="int8", speculative="ngram", num_speculative_tokens=4,
                              ngram_max_size=3, max_num_seqs=members, max_model_len=1700, kv_cache_memory_mb=64,
                              cuda_graphs=graphs, cuda_graph_max_batch=members, cuda_graph_max_context=1800,
                              prefix_cache=True, shared_prefix=shared)
    return create_verify_engine(CFG, state, settings, max_prefill_rows=640)


@pytest.mark.gpu
def test_verify_steps_read_a_cached_prompt_once():
    """70 requests on one cached prompt: steps from a captured graph give an eager engine's tokens,
    a step's hidden states are those of ordinary attention, and sharing ends with its reason."""
    state, members = unit_norms(), 70
    g = torch.Generator().manual_seed(9)
    prompt = torch.randint(0, 512, (16,), generator=g).tolist() * 96
    eager, graph, plain = (engine(state, members, *way).runner for way in ((True, False), (True, True), (False, False)))
    runs = {}
    for name, runner in (("eager", eager), ("graph", graph), ("plain", plain)):
        seqs = [Sequence.from_request(request(f"{i}", prompt + [i] * (i % 5), seed=i, ignore_eos=True,
                                              temperature=0.7 if i % 4 == 1 else 0.0)) for i in range(members)]
        runner.add(seqs[:1])
        assert not runner.sharing
        runner.add(seqs[1:])
        assert runner.sharing == (name != "plain")
        for _ in range(4):
            runner.step()
        runs[name] = [s.token_ids for s in seqs]
    assert runs["eager"] == runs["graph"] and graph.graph is not None and graph.graph_shared
    assert eager.model.workspace.error_flag() == 0 and graph.model.workspace.error_flag() == 0
    # the same step with and without: every real row's hidden state
    rows = members * eager.R
    real = (torch.arange(eager.R, device="cuda")[None, :] < eager.q_len[:, None]).flatten()
    both = []
    for batch in (eager.batch, eager.shared_batch):
        both.append(eager.model.forward(rows, eager.tokens, batch, eager.pool)[real].clone())
    assert real.sum() >= members and rel(both[1], both[0]) <= 2e-2
    # most requests end: sharing no longer pays, and the rest go on as the plain engine's would
    for runner in (eager, graph):
        for slot in range(3, members):
            runner.release(slot)
        assert not runner.sharing
        for _ in range(2):
            runner.step()
    assert [s.token_ids for s in eager.slots[:3]] == [s.token_ids for s in graph.slots[:3]] and not graph.graph_shared
    # and new requests on the prompt bring it back, in other slots' places
    more = [[Sequence.from_request(request(f"n{i}", prompt + [7, i], ignore_eos=True)) for i in range(members - 3)]
            for _ in range(2)]
    for runner, seqs in zip((eager, graph), more):
        runner.add(seqs)
        assert runner.sharing
        for _ in range(2):
            runner.step()
    assert [s.token_ids for s in more[0]] == [s.token_ids for s in more[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 1])
def test_requests_come_and_go_on_shared_blocks(seed, monkeypatch):
    """Random admissions, steps and releases of requests on nested prompts, every shared block read as one:
    the captured engine gives the eager one's tokens, and each step plans for the groups of that moment."""
    monkeypatch.setattr(kernels, "SHARED_PREFIX_MIN_BYTES", 1)
    state = unit_norms()
    g = torch.Generator().manual_seed(seed)
    trunk = torch.randint(0, 512, (16,), generator=g).tolist() * 14
    tails = [torch.randint(0, 512, (16,), generator=g).tolist() * n for n in (0, 3, 9)]
    runners = [engine(state, 9, True, graphs).runner for graphs in (False, True)]
    kept = [[], []]
    r = random.Random(seed)
    shared = 0
    for turn in range(40):
        op = r.choice(["add", "add", "step", "step", "step", "release"])
        free, busy = runners[0].free_slots(), runners[0].active_slots
        if op == "add" and free:
            n = r.randrange(1, len(free) + 1)
            made = [(f"{turn}.{i}", trunk + r.choice(tails) + [r.randrange(512) for _ in range(r.randrange(5))],
                     dict(temperature=r.choice([0.0, 0.9]), seed=r.randrange(99), ignore_eos=True)) for i in range(n)]
            for runner, all_of in zip(runners, kept):
                seqs = [Sequence.from_request(request(rid, list(tokens), **params)) for rid, tokens, params in made]
                all_of += seqs
                runner.add(seqs)
        elif op == "release" and busy:
            slot = r.choice(busy)
            for runner in runners:
                runner.release(slot)
        elif op == "step":
            for runner in runners:
                runner.step()
            shared += runners[0].sharing
        assert runners[0].active_slots == runners[1].active_slots and runners[0].sharing == runners[1].sharing
        assert [s.token_ids for s in kept[0]] == [s.token_ids for s in kept[1]]
    assert shared > 3 and all(runner.model.workspace.error_flag() == 0 for runner in runners)


@pytest.mark.gpu
def test_verification_refuses_filters_it_does_not_take():
    runner = engine(unit_norms(), 2, False, False).runner
    with pytest.raises(ValueError, match="top_k or min_p"):
        runner.add([Sequence.from_request(request("a", [1, 2], temperature=1.0, top_k=3))])
    assert runner.free_slots() == [0, 1]
    runner.add([Sequence.from_request(request("b", [1, 2], top_k=3))])  # greedy: nothing to filter
