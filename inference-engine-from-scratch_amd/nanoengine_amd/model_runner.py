"""One model step over a batch of sequences, in the reference's ModelRunner form.

Counterparts of ne/engine/generation/batch_builder.py:15-65 (``build_step_inputs``) and
ne/engine/generation/model_runner.py:14-80 (``ModelRunner.run_step`` / ``score_tokens``)
on the HIP forward (``Qwen3VerifyModel``).  The batched speculative loop does not come
through here: ``VerifyRunner`` packs its steps on the device.  This is the per-call seam
for callers of the reference's API, e.g. a speculative generator that scores one
sequence's guesses with ``score_tokens``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from nanoengine_amd import kernels
from nanoengine_amd.attention_context import AttentionContext, build_attention_mask
from nanoengine_amd.interface import GREEDY_TEMPERATURE, GenerationRequest, sampling_uniform
from nanoengine_amd.memory import find_shared_prefixes
from nanoengine_amd.qwen3 import AttentionBatch, Qwen3VerifyModel
from nanoengine_amd.sequence_state import Sequence

PADDING_TOKEN_ID = 0
# A shared-prefix plan has room for the longest sequence's queries in every sequence: 64 sequences of which
# one brings 1,024 queries would hold 1.1 GB of partial sums.  Past this many bytes a step of which more
# than half is padding takes ordinary attention.
SHARED_PREFIX_MAX_PADDED = 256 << 20


@dataclass(frozen=True)
class StepInputs:
    token_ids: torch.Tensor  # [b, q]
    context: AttentionContext
    last_token_indices: torch.Tensor  # [b] index of each sequence's last real token in q


def build_step_inputs(sequences: list, allocator, pool, device: torch.device,
                      token_counts: list[int] | None = None) -> StepInputs:
    """Each sequence brings its next ``token_counts[i]`` uncached tokens (default: all of
    them), padded to the longest; padding rows write to the pool's scratch slot.  The
    context also carries the block tables, real-row counts and context lengths the paged
    kernels read.  KV memory for the new tokens must already be reserved."""
    counts = token_counts or [s.num_uncached_tokens for s in sequences]
    ends = [s.num_cached_tokens + n for s, n in zip(sequences, counts, strict=True)]
    q = max(counts)
    c = max(ends)
    token_rows, position_rows = [], []
    for s, end in zip(sequences, ends, strict=True):
        start = s.num_cached_tokens
        pad = [PADDING_TOKEN_ID] * (q - (end - start))
        token_rows.append(s.token_ids[start:end] + pad)
        position_rows.append(list(range(start, end)) + pad)
    token_ids = torch.tensor(token_rows, device=device)
    positions = torch.tensor(position_rows, device=device)
    n = torch.tensor(counts, device=device)
    is_real = torch.arange(q, device=device)[None, :] < n[:, None]
    context_slots = allocator.build_context_slots(sequences, c)
    slot_mapping = context_slots.gather(1, positions).masked_fill(~is_real, pool.scratch_slot)
    context_lengths = torch.tensor(ends, device=device)
    blocks = math.ceil(c / pool.block_size)
    tables = [(allocator.block_table(s)[:blocks] + [0] * blocks)[:blocks] for s in sequences]
    context = AttentionContext(
        positions=positions,
        slot_mapping=slot_mapping,
        context_slots=context_slots,
        attention_mask=build_attention_mask(positions, context_lengths, c),
        key_caches=pool.key_caches,
        value_caches=pool.value_caches,
        key_scales=pool.key_scales,
        value_scales=pool.value_scales,
        block_tables=torch.tensor(tables, dtype=torch.int32, device=device),
        block_size=pool.block_size,
        query_lengths=n.to(torch.int32),
        context_lengths=context_lengths.to(torch.int32),
        max_context_length=c,
    )
    return StepInputs(token_ids=token_ids, context=context, last_token_indices=n - 1)


class ModelRunner:
    """Runs the HIP forward for padded steps of a few sequences (model_runner.py:14-80).

    ``shared_prefix`` lets a step read the blocks that its sequences share (a prefix cache's, or
    those of :meth:`fork`) once for all of them, where that pays."""

    def __init__(self, model: Qwen3VerifyModel, pool, allocator, device: torch.device,
                 shared_prefix: bool = False) -> None:
        self.shared_prefix = shared_prefix
        self._model = model
        self._pool = pool
        self.allocator = allocator
        self._device = device

    @property
    def vocab_size(self) -> int:
        return self._model.config.vocab_size

    def _prefix_groups(self, sequences: list, counts: list[int], max_ctx_len: int) -> kernels.PrefixGroups | None:
        """The sequences' groups, if this step's attention is to read their prefixes once."""
        pool = self._pool
        if len(sequences) > kernels.SHARED_PREFIX_MAX_SEQS or not kernels.shared_prefix_supported(
                pool.key_caches[0], None if pool.key_scales is None else pool.key_scales[0]):
            return None
        c, size = self._model.config, pool.block_size
        found = find_shared_prefixes([self.allocator.block_table(s) for s in sequences])
        saved = sum((len(members) - 1) * blocks * size for members, blocks in found)
        if not kernels.shared_prefix_pays(saved, c.num_key_value_heads, pool.key_caches[0].dtype):
            return None
        grouped = {i for members, _ in found for i in members}
        singles = [i for i in range(len(sequences)) if i not in grouped]
        nbytes = kernels.shared_prefix_workspace_bytes(
            len(sequences), len(found) + len(singles), c.num_attention_heads, c.num_key_value_heads, max(counts),
            max_ctx_len, max(blocks for _, blocks in found) * size)
        padded = len(counts) * max(counts) > 2 * sum(counts)
        if nbytes == 0 or padded and nbytes > SHARED_PREFIX_MAX_PADDED:  # (0: a shape that no plan is made for)
            return None
        return kernels.PrefixGroups.from_lists([members for members, _ in found] + [[i] for i in singles],
                                               [blocks * size for _, blocks in found] + [0] * len(singles),
                                               self._device)

    def fork(self, sequence: Sequence, request: GenerationRequest) -> Sequence:
        """A new sequence for ``request``, whose prompt starts with ``sequence``'s cached tokens:
        it begins with their keys and values (all, or but the prompt's last token, which a step
        has to compute), shared where the allocator shares blocks and copied otherwise."""
        child = Sequence.from_request(request)
        shared = min(sequence.num_cached_tokens, child.num_tokens - 1)
        if shared < 0 or child.token_ids[:shared] != sequence.token_ids[:shared]:
            raise ValueError(f"{child.request_id} does not start with the cached tokens of {sequence.request_id}")
        src, dst = self.allocator.fork(sequence, child, shared)
        try:
            self._pool.copy_blocks(src, dst)
        except BaseException:
            self.allocator.free(child)
            raise
        child.num_cached_tokens = shared
        return child

    def _forward(self, inputs: StepInputs, sequences: list):
        """The step's real rows packed sequence after sequence, through the model; returns
        the hidden states and each sequence's first row."""
        ctx = inputs.context
        counts = ctx.query_lengths.tolist()
        q = inputs.token_ids.shape[1]
        real = torch.arange(q, device=self._device)[None, :] < ctx.query_lengths[:, None].long()
        tokens = inputs.token_ids[real].to(torch.int32)
        starts = [0]
        for n in counts[:-1]:
            starts.append(starts[-1] + n)
        batch = AttentionBatch(
            positions=ctx.positions[real].to(torch.int32),
            slot_mapping=ctx.slot_mapping[real].to(torch.int32),
            q_start=torch.tensor(starts, dtype=torch.int32, device=self._device),
            q_len=ctx.query_lengths,
            ctx_len=ctx.context_lengths,
            block_tables=ctx.block_tables,
            max_q_len=max(counts),
            max_ctx_len=ctx.max_context_length,
            prefix_groups=self._prefix_groups(sequences, counts, ctx.max_context_length) if self.shared_prefix else None,
        )
        rows = sum(counts)
        if rows > self._model.max_rows:
            raise ValueError(f"{rows} rows exceed the model's capacity of {self._model.max_rows}; "
                             "pass smaller token_counts (chunked prefill)")
        self._model.ensure_rope(ctx.max_context_length)
        hidden = self._model.forward(rows, tokens, batch, self._pool, workspace=self._model.eager_workspace)
        return hidden, starts, counts

    @torch.inference_mode()
    def score_tokens(self, sequence, token_count: int) -> torch.Tensor:
        """Cache the next ``token_count`` tokens of one sequence and return the logits after
        each of them, ``[token_count, vocab]`` bf16 (model_runner.py:52-62)."""
        inputs = build_step_inputs([sequence], self.allocator, self._pool, self._device, [token_count])
        hidden, _, _ = self._forward(inputs, [sequence])
        sequence.num_cached_tokens += token_count
        self.allocator.on_tokens_cached(sequence)
        logits, _ = self._model.compute_logits(hidden[:token_count])
        return logits

    def _draw_filtered(self, logits: torch.Tensor, sequences: list) -> torch.Tensor:
        params = [s.sampling_params for s in sequences]
        streams = [s.sampling_generator for s in sequences]

        def row(values, dtype=torch.float32):
            return torch.tensor(values, dtype=dtype, device=self._device)

        return kernels.sample(
            logits, row([sampling_uniform(s.seed, s.step) for s in streams]),
            temperature=row([p.temperature for p in params]),
            top_k=row([min(max(p.top_k, 0), self.vocab_size) for p in params], torch.int32),
            top_p=row([p.top_p for p in params]), min_p=row([p.min_p for p in params]))

    def _accept_last(self, logits: torch.Tensor, sequences: list) -> torch.Tensor:
        """Each row's token by the acceptance kernel, as a verify step without guesses."""
        b = len(sequences)
        params = [s.sampling_params for s in sequences]
        drafts = torch.zeros((b, 1), dtype=torch.int32, device=self._device)
        no_drafts = torch.zeros((b,), dtype=torch.int32, device=self._device)
        row_start = torch.arange(b, dtype=torch.int32, device=self._device)
        kwargs = {}
        if any(p.temperature != GREEDY_TEMPERATURE for p in params):
            kwargs = dict(
                temperature=torch.tensor([p.temperature for p in params], dtype=torch.float32, device=self._device),
                top_p=torch.tensor([p.top_p for p in params], dtype=torch.float32, device=self._device),
                seeds=torch.tensor([s.sampling_generator.seed for s in sequences], dtype=torch.int64,
                                   device=self._device),
                steps=torch.tensor([s.sampling_generator.step for s in sequences], dtype=torch.int64,
                                   device=self._device),
                any_sampled=True,
            )
        out, _ = kernels.accept(drafts, no_drafts, row_start, self.vocab_size, logits=logits, **kwargs)
        return out[:, 0]

    @torch.inference_mode()
    def run_step(self, sequences: list, token_counts: list[int] | None = None) -> list[int]:
        """Cache the next ``token_counts`` tokens of each sequence (default: all uncached)
        and pick a token after each one's last (model_runner.py:33-50): the argmax, or for a
        sampled request a draw under the explicit-uniform contract of the acceptance kernel
        at the request's temperature and top-p, advancing its sampling stream.  A request that
        also has a top-k or min-p gets the token that ``kernels.sample`` draws, from the
        stream's uniform of its own at each step."""
        inputs = build_step_inputs(sequences, self.allocator, self._pool, self._device, token_counts)
        hidden, starts, counts = self._forward(inputs, sequences)
        last = torch.tensor([s + n - 1 for s, n in zip(starts, counts, strict=True)], device=self._device)
        logits, _ = self._model.compute_logits(hidden[last].contiguous())
        filtered = [i for i, s in enumerate(sequences) if s.sampling_params.is_filtered]
        if len(filtered) == len(sequences):
            tokens = self._draw_filtered(logits, sequences).tolist()
        else:
            out = self._accept_last(logits, sequences)
            if filtered:
                out[filtered] = self._draw_filtered(logits[filtered], [sequences[i] for i in filtered])
            tokens = out.tolist()
        for s in sequences:
            if s.sampling_params.temperature != GREEDY_TEMPERATURE:
                s.sampling_generator.step += 1
        final_counts = token_counts or counts
        for s, n in zip(sequences, final_counts, strict=True):
            s.num_cached_tokens += n
            self.allocator.on_tokens_cached(s)
        return tokens
