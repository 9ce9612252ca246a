"""Operators of serving many answers to one prompt, case by case, with their plain forms.

A case is a dict of plain values; ``kind`` says which operator it runs:

  copy       copying KV blocks of every layer's caches within a pool (a fork's partial
             blocks, whole prompts)
  attention  attention of a batch whose sequences share prefixes: one work plan, then the
             attention of several layers' pools, as a step runs them
  sample     a token per row of logits from a given uniform, under temperature, top-k,
             top-p and min-p; with ``probs`` the filtered distribution too

``own`` selects what ``run`` calls: the plain forms here (elementary torch operations in
32 bits, in 64 where a value next to a border decides a token), or the library's kernels.
Lengths are spread evenly between a case's bounds and dealt to the sequences in an order
drawn from the seed, so the work of a case does not depend on the seed.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

HEAD = 128
VOCAB = 151936
SCALE = 1.0 / math.sqrt(HEAD)


def _kernels():
    package = str(Path(__file__).resolve().parents[1] / "inference-engine-from-scratch_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nanoengine_amd import kernels

    return kernels


# ------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # eight samples of one prompt: seven copies of its last, partly filled block (latency)
        {"name": "copy_tails_7_bf16", "kind": "copy", "kv": "bf16", "layers": 28, "heads": 8, "block": 16,
         "blocks": 256, "pairs": 7},
        # 64 prompts of 256 tokens moved whole, int8 pool (half the 0.6B model's layers)
        {"name": "copy_1024_int8", "kind": "copy", "kv": "int8", "layers": 14, "heads": 8, "block": 16,
         "blocks": 2500, "pairs": 1024},
        # four samples of one request, one new token each
        {"name": "prefix_decode_4x1_bf16", "kind": "attention", "kv": "bf16", "layers": 4, "q_heads": 16,
         "kv_heads": 8, "block": 16, "groups": 1, "seqs": 4, "q_lo": 1, "q_hi": 1, "prefix_lo": 544,
         "prefix_hi": 544, "suffix_lo": 1, "suffix_hi": 40},
        # a batched verify step under one system prompt: 64 sequences, four guesses each
        {"name": "prefix_verify_64x5_int8", "kind": "attention", "kv": "int8", "layers": 4, "q_heads": 16,
         "kv_heads": 8, "block": 16, "groups": 1, "seqs": 64, "q_lo": 5, "q_hi": 5, "prefix_lo": 1024,
         "prefix_hi": 1024, "suffix_lo": 16, "suffix_hi": 256},
        # 64 samples over a long document
        {"name": "prefix_decode_64x1_long_bf16", "kind": "attention", "kv": "bf16", "layers": 2, "q_heads": 16,
         "kv_heads": 8, "block": 16, "groups": 1, "seqs": 64, "q_lo": 1, "q_hi": 1, "prefix_lo": 16384,
         "prefix_hi": 16384, "suffix_lo": 64, "suffix_hi": 1024},
        # several prompts with samples of their own, ragged guesses, prefixes that end inside a tile
        {"name": "prefix_groups_7_ragged_int8", "kind": "attention", "kv": "int8", "layers": 2, "q_heads": 16,
         "kv_heads": 8, "block": 16, "groups": 7, "seqs": 45, "q_lo": 1, "q_hi": 9, "prefix_lo": 112,
         "prefix_hi": 4000, "suffix_lo": 1, "suffix_hi": 700},
        # the long-context verify step: 32 sequences on a 1,024-token prefix, eight guesses each
        {"name": "prefix_verify_32x9_long_int8", "kind": "attention", "kv": "int8", "layers": 2, "q_heads": 16,
         "kv_heads": 8, "block": 16, "groups": 1, "seqs": 32, "q_lo": 9, "q_hi": 9, "prefix_lo": 1024,
         "prefix_hi": 1024, "suffix_lo": 4096, "suffix_hi": 16384},
        # one request's next token, every filter on (latency)
        {"name": "sample_1_filters", "kind": "sample", "rows": 1, "vocab": VOCAB, "dtype": "bf16",
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02, "each": False, "probs": False},
        # a batch of requests with parameters of their own, greedy ones among them
        {"name": "sample_64_each_its_own", "kind": "sample", "rows": 64, "vocab": VOCAB, "dtype": "bf16",
         "temperature": 0.9, "top_k": 400, "top_p": 0.9, "min_p": 0.05, "each": True, "probs": False},
        # 64 sequences' five guesses with the distributions that a verifier reads
        {"name": "sample_320_top_p_probs", "kind": "sample", "rows": 320, "vocab": VOCAB, "dtype": "bf16",
         "temperature": 0.8, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "each": False, "probs": True},
        # 32-bit logits of a small, odd vocabulary, temperature alone
        {"name": "sample_200_plain_fp32", "kind": "sample", "rows": 200, "vocab": 32003, "dtype": "fp32",
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "each": False, "probs": False},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["copy", "attention", "attention", "sample", "sample"])
    if kind == "copy":
        kv = rng.choice(["bf16", "int8"])
        pairs = _log(rng, 1, 1000)
        return {"kind": kind, "kv": kv, "layers": rng.randint(1, 28 if kv == "bf16" else 14),
                "heads": rng.choice([2, 4, 8]), "block": rng.choice([16, 32]),
                "blocks": 2 * pairs + rng.randint(1, 99), "pairs": pairs}
    if kind == "attention":
        groups = rng.choice([1, 1, 2, 5, 9])
        kv_heads, ratio = rng.choice([(8, 2), (8, 2), (8, 4), (4, 2), (2, 8)])
        prefix, suffix = _log(rng, 32, 12000), _log(rng, 2, 3000)
        q = rng.choice([1, 1, 3, 5, 9])
        return {"kind": kind, "kv": rng.choice(["bf16", "int8"]), "layers": rng.randint(1, 3),
                "q_heads": kv_heads * ratio, "kv_heads": kv_heads, "block": rng.choice([16, 16, 32]),
                "groups": groups, "seqs": groups + _log(rng, 1, 60), "q_lo": rng.randint(1, q), "q_hi": q,
                "prefix_lo": rng.randint(max(1, prefix // 4), prefix), "prefix_hi": prefix,
                "suffix_lo": rng.randint(1, suffix), "suffix_hi": suffix}
    rows = _log(rng, 1, 300)
    return {"kind": kind, "rows": rows, "vocab": _log(rng, 500, VOCAB), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "temperature": round(rng.uniform(0.4, 1.5), 2), "top_k": rng.choice([0, 1, 20, 50, _log(rng, 2, 5000)]),
            "top_p": rng.choice([1.0, 0.5, 0.9, 0.95]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
            "each": rng.random() < 0.5, "probs": rng.random() < 0.3}


# ------------------------------------------------------------------------ lengths and work
def _spread(lo: int, hi: int, n: int) -> list[int]:
    """``n`` numbers spread evenly from ``lo`` to ``hi``."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _members(case: dict) -> list[int]:
    """Sequences of each group: one each, the rest in shares that fall with the group's number."""
    g, rest = case["groups"], case["seqs"] - case["groups"]
    weights = [g - i for i in range(g)]
    counts = [1 + rest * w // sum(weights) for w in weights]
    counts[0] += case["seqs"] - sum(counts)
    return counts


def _prefixes(case: dict) -> list[int]:
    """Shared tokens of each group: whole blocks, as a prefix cache shares them."""
    return [p // case["block"] * case["block"] for p in _spread(case["prefix_lo"], case["prefix_hi"], case["groups"])]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, tokens after the prefix before them) of each sequence, before the seed deals them."""
    n = case["seqs"]
    return _spread(case["q_lo"], case["q_hi"], n), _spread(case["suffix_lo"], case["suffix_hi"], n)


def _order(count: int, step: int) -> list[int]:
    """A fixed order of the sequences that pairs unlike lengths, the same for every seed."""
    while math.gcd(step, count) != 1:
        step += 1
    return [(i * step) % count for i in range(count)]


def _sequences(case: dict) -> list[tuple[int, int, int]]:
    """(group, new tokens, suffix tokens before them) of every sequence, in group order."""
    q, suffix = _lengths(case)
    a, b = _order(case["seqs"], 7), _order(case["seqs"], 11)
    groups = [g for g, c in enumerate(_members(case)) for _ in range(c)]
    return [(g, q[a[i]], suffix[b[i]]) for i, g in enumerate(groups)]


def _slot_bytes(kv: str, heads: int) -> int:
    return heads * (HEAD + 2) if kv == "int8" else heads * HEAD * 2


def work(case: dict) -> dict:
    if case["kind"] == "copy":
        moved = case["pairs"] * case["block"] * 2 * case["layers"] * _slot_bytes(case["kv"], case["heads"])
        return {"bytes": 2 * moved, "flops": 0}
    if case["kind"] == "attention":
        prefixes = _prefixes(case)
        seqs = _sequences(case)
        slots = sum(prefixes) + sum(s + q for _, q, s in seqs)
        rows = sum(q for _, q, _ in seqs)
        seen = sum(q * (prefixes[g] + s) + q * (q + 1) // 2 for g, q, s in seqs)
        per_layer = slots * 2 * _slot_bytes(case["kv"], case["kv_heads"]) + 2 * rows * case["q_heads"] * HEAD * 2
        return {"bytes": case["layers"] * per_layer, "flops": case["layers"] * 4 * HEAD * case["q_heads"] * seen}
    size = case["rows"] * case["vocab"]
    element = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": size * (element + (4 if case["probs"] else 0)) + 8 * case["rows"], "flops": 4 * size}


# ------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _caches(kv: str, layers: int, slots: int, heads: int, g: torch.Generator) -> dict:
    """Per-layer caches ``[slots, heads, 128]`` in the pool's layout; int8 ones with scales ``[slots, heads]``."""
    shape = (slots, heads, HEAD)
    if kv == "int8":
        code = lambda: torch.randint(-127, 128, shape, device="cuda", dtype=torch.int8, generator=g)
        scale = lambda: (0.012 + 0.02 * torch.rand((slots, heads), device="cuda", generator=g)).to(torch.bfloat16)
        return {"k": [code() for _ in range(layers)], "v": [code() for _ in range(layers)],
                "ks": [scale() for _ in range(layers)], "vs": [scale() for _ in range(layers)]}
    value = lambda: torch.randn(shape, device="cuda", dtype=torch.bfloat16, generator=g)
    return {"k": [value() for _ in range(layers)], "v": [value() for _ in range(layers)],
            "ks": [None] * layers, "vs": [None] * layers}


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    rng = np.random.default_rng(seed)
    if case["kind"] == "copy":
        caches = _caches(case["kv"], case["layers"], case["blocks"] * case["block"] + 1, case["heads"], g)
        blocks = rng.permutation(case["blocks"])
        return {"case": case, "buffers": [t for name in ("k", "v", "ks", "vs") for t in caches[name] if t is not None],
                "src": blocks[: case["pairs"]].tolist(), "dst": blocks[case["pairs"] : 2 * case["pairs"]].tolist()}
    if case["kind"] == "attention":
        return _prepare_attention(case, g, rng)
    shape = (case["rows"], case["vocab"])
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
    # a language model's logits: a broad bulk and some tens of likely tokens above it
    logits = 2.0 * torch.randn(shape, device="cuda", generator=g)
    likely = torch.randint(0, case["vocab"], (case["rows"], 40), device="cuda", generator=g)
    logits.scatter_add_(1, likely, 4.0 + 8.0 * torch.rand((case["rows"], 40), device="cuda", generator=g))
    state = {"case": case, "logits": logits.to(dtype),
             "u": torch.rand(case["rows"], device="cuda", generator=g)}
    if case["each"]:  # every request's own parameters; one in eight is greedy
        vary = torch.rand((4, case["rows"]), device="cuda", generator=g)
        greedy = torch.arange(case["rows"], device="cuda") % 8 == 7
        state["temperature"] = (case["temperature"] * (0.5 + vary[0])).masked_fill(greedy, 0.0)
        state["top_k"] = (case["top_k"] * 2 * vary[1]).to(torch.int32)
        state["top_p"] = case["top_p"] + (1.0 - case["top_p"]) * vary[2]
        state["min_p"] = case["min_p"] * 2 * vary[3]
    else:
        state |= {name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")}
    return state


def _prepare_attention(case: dict, g: torch.Generator, rng) -> dict:
    bs, n = case["block"], case["seqs"]
    prefixes, seqs = _prefixes(case), _sequences(case)
    place = rng.permutation(n)  # a group's members sit in any slots of the batch
    need = sum(p // bs for p in prefixes) + sum((s + q + bs - 1) // bs for _, q, s in seqs)
    pool = need + 37
    blocks = rng.permutation(pool)
    shared, at = [], 0
    for p in prefixes:
        shared.append(blocks[at : at + p // bs])
        at += p // bs
    ctx, q_len = np.zeros(n, np.int32), np.zeros(n, np.int32)
    width = max((prefixes[k] + s + q + bs - 1) // bs for k, q, s in seqs)
    tables = np.zeros((n, width), np.int32)
    for i, (k, q, s) in enumerate(seqs):
        slot, extra = place[i], (s + q + bs - 1) // bs
        ctx[slot], q_len[slot] = prefixes[k] + s + q, q
        tables[slot, : len(shared[k])] = shared[k]
        tables[slot, len(shared[k]) : len(shared[k]) + extra] = blocks[at : at + extra]
        at += extra
    counts = _members(case)
    rows = int(q_len.sum())
    q_start = np.concatenate([[0], np.cumsum(q_len)[:-1]]).astype(np.int32)
    dev = lambda x, dtype=np.int32: torch.from_numpy(np.ascontiguousarray(x, dtype)).cuda()
    caches = _caches(case["kv"], case["layers"], pool * bs + 1, case["kv_heads"], g)
    return {"case": case, **caches,
            "q": [1.5 * torch.randn((rows, case["q_heads"], HEAD), device="cuda", dtype=torch.bfloat16, generator=g)
                  for _ in range(case["layers"])],
            "tables": dev(tables), "ctx": dev(ctx), "q_start": dev(q_start), "q_len": dev(q_len),
            "group_seqs": dev(place), "group_start": dev(np.concatenate([[0], np.cumsum(counts)])),
            "prefix_len": dev(prefixes), "max_q": int(q_len.max()), "max_ctx": int(ctx.max()),
            "max_prefix": max(prefixes), "max_members": max(counts),
            "max_suffix": max(s + q for _, q, s in seqs)}


# ------------------------------------------------------------------------ a pass
def run(state: dict):
    case = state["case"]
    if case["kind"] == "copy":
        if own:
            _kernels().copy_kv_blocks(state["buffers"], case["block"], state["src"], state["dst"])
        else:
            _copy_plain(state)
        return state["buffers"]
    if case["kind"] == "attention":
        if own:
            return _attention_own(state)
        return [_attention_plain(state, i) for i in range(case["layers"])]
    if own:
        return _kernels().sample(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"], probs=case["probs"])
    return _sample_plain(state)


def _attention_own(s: dict):
    kernels, case = _kernels(), s["case"]
    groups = kernels.PrefixGroups(s["group_seqs"], s["group_start"], s["prefix_len"], s["max_prefix"])
    plan = kernels.shared_prefix_plan(s["tables"], case["block"], s["ctx"], s["q_start"], s["q_len"], groups,
                                      case["q_heads"], case["kv_heads"], s["max_q"], s["max_ctx"])
    return [kernels.shared_prefix_attention(s["q"][i], s["k"][i], s["v"][i], s["ks"][i], s["vs"][i], plan)
            for i in range(case["layers"])]


def _copy_plain(s: dict) -> None:
    bs = s["case"]["block"]
    src = torch.tensor(s["src"], device="cuda")
    dst = torch.tensor(s["dst"], device="cuda")
    for buffer in s["buffers"]:
        blocks = buffer[: s["case"]["blocks"] * bs].view(s["case"]["blocks"], bs, -1)
        blocks[dst] = blocks[src]


def _vectors(cache: torch.Tensor, scale: torch.Tensor | None, slots: torch.Tensor) -> torch.Tensor:
    """fp32 head vectors ``[.., kv_heads, keys, 128]`` of the slots ``[.., keys]``."""
    x = cache[slots].float()
    if scale is not None:
        x = x * scale[slots].float().unsqueeze(-1)
    return x.transpose(-2, -3).contiguous()


def _attention_plain(s: dict, layer: int) -> torch.Tensor:
    """The prefix's scores and values once per group, the rest per sequence, one softmax over both."""
    case = s["case"]
    bs, heads = case["block"], case["kv_heads"]
    ratio = case["q_heads"] // heads
    n, mq = case["seqs"], s["max_q"]
    tables, ctx, q_len = s["tables"].long(), s["ctx"].long(), s["q_len"].long()
    dev = tables.device
    start = s["group_start"].long()
    members = torch.arange(s["max_members"], device=dev)
    entry = start[:-1, None] + members  # [G, M]
    inside = entry < start[1:, None]
    who = s["group_seqs"].long()[entry.clamp(max=n - 1)]  # [G, M] sequences
    prefix = s["prefix_len"].long()
    group_of = torch.zeros(n, dtype=torch.long, device=dev)
    member_of = torch.zeros(n, dtype=torch.long, device=dev)
    g_index = torch.arange(case["groups"], device=dev)[:, None].expand_as(who)
    group_of[who[inside]] = g_index[inside]
    member_of[who[inside]] = members.expand_as(who)[inside]

    i = torch.arange(mq, device=dev)
    row = (s["q_start"].long()[:, None] + i).clamp(max=s["q"][layer].shape[0] - 1)  # [n, mq]
    real = i < q_len[:, None]
    q = s["q"][layer].float()[row].view(n, mq, heads, ratio, HEAD).permute(0, 2, 1, 3, 4)
    q = q.reshape(n, heads, mq * ratio, HEAD).contiguous()  # rows (query, head of the group)

    def slots_of(table, key):
        return table.gather(1, (key // bs).clamp(max=table.shape[1] - 1)) * bs + key % bs

    # keys 0 .. P-1, once per group
    key_p = torch.arange(s["max_prefix"], device=dev).expand(case["groups"], -1)
    slots_p = slots_of(tables[who[:, 0]], key_p)
    k_p = _vectors(s["k"][layer], s["ks"][layer], slots_p)
    v_p = _vectors(s["v"][layer], s["vs"][layer], slots_p)
    q_g = q[who].transpose(1, 2).reshape(case["groups"], heads, -1, HEAD).contiguous()  # [G, heads, M * mq * ratio, 128]
    s_p = torch.matmul(q_g, k_p.transpose(-1, -2).contiguous()) * SCALE
    s_p = s_p.masked_fill((key_p >= prefix[:, None])[:, None, None, :], -math.inf)
    # keys P .. of every sequence
    own_prefix = prefix[group_of]
    key_s = own_prefix[:, None] + torch.arange(s["max_suffix"], device=dev)
    slots_s = slots_of(tables, key_s)
    k_s = _vectors(s["k"][layer], s["ks"][layer], slots_s)
    v_s = _vectors(s["v"][layer], s["vs"][layer], slots_s)
    position = ctx[:, None] - q_len[:, None] + i  # [n, mq]
    hidden = (key_s[:, None, :] > position[:, :, None]) | ~real[:, :, None]  # [n, mq, S]
    s_s = torch.matmul(q, k_s.transpose(-1, -2).contiguous()) * SCALE
    s_s = s_s.masked_fill(hidden.repeat_interleave(ratio, 1)[:, None], -math.inf)

    def to_group(x):  # [n, heads, R, ..] -> [G, heads, M * R, ..]
        return x[who].transpose(1, 2).reshape(case["groups"], heads, -1, x.shape[-1])

    def to_seq(x):  # [G, heads, M * R, ..] -> [n, heads, R, ..]
        x = x.view(case["groups"], heads, -1, mq * ratio, x.shape[-1])
        return x[group_of, :, member_of]

    top = torch.maximum(to_seq(s_p.amax(-1, keepdim=True)), s_s.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    e_p = torch.exp(s_p - to_group(top))
    e_s = torch.exp(s_s - top)
    total = to_seq(e_p.sum(-1, keepdim=True)) + e_s.sum(-1, keepdim=True)
    o = to_seq(torch.matmul(e_p, v_p)) + torch.matmul(e_s, v_s)
    o = (o / total).view(n, heads, mq, ratio, HEAD).permute(0, 2, 1, 3, 4).reshape(n, mq, heads * ratio, HEAD)
    out = torch.empty_like(s["q"][layer])
    out[row[real]] = o[real].to(torch.bfloat16)
    return out


def _sample_plain(s: dict):
    """In 64 bits: a uniform next to a border between two tokens decides between them."""
    rows, vocab = s["logits"].shape

    def column(x):
        x = x if isinstance(x, torch.Tensor) else torch.full((rows,), x, device="cuda", dtype=torch.float32)
        return x.double()[:, None]

    temperature, top_k, top_p, min_p = (column(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    x, index = s["logits"].double().sort(dim=1, descending=True, stable=True)
    greedy = temperature == 0.0
    z = (x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature)
    w = torch.exp(z)
    rank = torch.arange(vocab, device="cuda", dtype=torch.float64)
    keep = (rank < top_k) | (top_k <= 0)
    w = w * keep
    before = w.cumsum(1) - w
    keep &= (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1.0)
    keep &= w >= min_p
    keep = torch.where(greedy, rank < 1, keep) | (rank < 1)
    w = w * keep
    running = w.cumsum(1)
    total = w.sum(1, keepdim=True)
    chosen = (running <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    chosen = torch.minimum(chosen, keep.sum(1, keepdim=True) - 1)
    token = index.gather(1, chosen).squeeze(1).to(torch.int32)
    if not s["case"]["probs"]:
        return token
    return token, torch.zeros_like(w).scatter_(1, index, w / total).float()


# ------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    if case["kind"] == "copy":
        return None  # copies: no computed numbers
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return [_attention_exact(s, i) for i in range(case["layers"])]
    if not case["probs"]:
        return None  # a token a row: whole numbers
    return None, _probs_exact(s)


def _attention_exact(s: dict, layer: int) -> torch.Tensor:
    """Every sequence by itself over its whole context."""
    case = s["case"]
    heads, bs = case["kv_heads"], case["block"]
    out = torch.empty(s["q"][layer].shape, dtype=torch.float64, device="cuda")
    lists = [s[name].tolist() for name in ("ctx", "q_start", "q_len")]
    for b, (ctx, start, count) in enumerate(zip(*lists)):
        p = torch.arange(ctx, device="cuda")
        slot = s["tables"][b].long()[p // bs] * bs + p % bs
        k, v = s["k"][layer][slot].double(), s["v"][layer][slot].double()
        if case["kv"] == "int8":
            k = k * s["ks"][layer][slot].double()[..., None]
            v = v * s["vs"][layer][slot].double()[..., None]
        q = s["q"][layer][start : start + count].double().view(count, heads, -1, HEAD)
        score = (q.permute(1, 2, 0, 3).reshape(heads, -1, HEAD) @ k.permute(1, 2, 0).contiguous()) / math.sqrt(HEAD)
        score = score.view(heads, -1, count, ctx)
        position = ctx - count + torch.arange(count, device="cuda")
        score = score.masked_fill(p > position[:, None], -math.inf)
        prob = torch.softmax(score, -1).reshape(heads, -1, ctx)
        o = (prob @ v.permute(1, 0, 2).contiguous()).view(heads, -1, count, HEAD)
        out[start : start + count] = o.permute(2, 0, 1, 3).reshape(count, -1, HEAD)
    return out


def _probs_exact(s: dict) -> torch.Tensor:
    """The filtered distribution of every row from its own numbers, on the host."""
    x = s["logits"].double().cpu().numpy()
    rows, vocab = x.shape
    value = lambda name, r: float(s[name][r]) if isinstance(s[name], torch.Tensor) else float(np.float32(s[name]))
    out = np.zeros((rows, vocab))
    for r in range(rows):
        t, k, p, m = (value(name, r) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-x[r], kind="stable")
        if t == 0.0:
            out[r, order[0]] = 1.0
            continue
        w = np.exp((x[r, order] - x[r, order[0]]) / t)
        n = vocab if k <= 0 else min(int(k), vocab)
        mass = np.cumsum(w[:n])
        if p < 1.0:
            n = min(n, 1 + int(np.searchsorted(mass, p * mass[-1], side="left")))
        n = max(1, min(n, int(np.count_nonzero(w >= m))))
        out[r, order[:n]] = w[:n] / w[:n].sum()
    return torch.from_numpy(out).cuda()
