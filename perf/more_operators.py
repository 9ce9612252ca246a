"""Operators of a step on both ends of a model, case by case, with their plain forms.

A case is a dict of plain values; ``kind`` says which operator it runs:

  product    rows of activations to 8-bit integers with a scale per row (``norm``: through
             RMSNorm), then their product with 8-bit weights of a scale per output column;
             ``swiglu``: gate and up columns paired per 16, bf16(silu(gate) * up)
  adjust     logits under repetition, presence and frequency penalties for the tokens of each
             row's history (and the guesses before it in a verify step), biases of single
             tokens, and bit masks of allowed tokens

``own`` selects what ``run`` calls: the plain forms here (elementary torch operations in
32 bits, in 64 where a quotient next to a half decides a code), or the library's kernels.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

VOCAB = 151936
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kernels():
    package = str(Path(__file__).resolve().parents[1] / "inference-engine-from-scratch_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nanoengine_amd import kernels

    return kernels


# ------------------------------------------------------------------------ the cases
def _product(name, m, n, k, norm=False, swiglu=False, dtype="bf16", scale="bf16") -> dict:
    return {"name": name, "kind": "product", "m": m, "n": n, "k": k, "norm": norm, "swiglu": swiglu, "dtype": dtype,
            "scale": scale}


def _adjust(name, seqs, guesses, len_lo, len_hi, bias, masks, penalties=True, vocab=VOCAB, dtype="bf16", out="bf16") -> dict:
    return {"name": name, "kind": "adjust", "seqs": seqs, "guesses": guesses, "len_lo": len_lo, "len_hi": len_hi, "bias": bias,
            "masks": masks, "penalties": penalties, "vocab": vocab, "dtype": dtype, "out": out}


def listed() -> list[dict]:
    return [
        # one request's next token: its q, k and v (latency)
        _product("product_1_qkv", 1, 4096, 1024, norm=True),
        # a batch's next tokens: the attention output's projection
        _product("product_64_o", 64, 1024, 2048),
        # a short prompt: gate and up, an odd number of rows
        _product("product_333_swiglu", 333, 6144, 1024, norm=True, swiglu=True),
        # a batch's logits: the output head in 8 bits, the weights' stream
        _product("product_64_head", 64, VOCAB, 1024, norm=True),
        # prompts of a few thousand tokens, ragged
        _product("product_4001_o", 4001, 1024, 2048),
        # a chunk of a long prompt: q, k and v
        _product("product_8192_qkv", 8192, 4096, 1024, norm=True),
        # a larger model's square projection, fp16 activations and fp32 scales
        _product("product_8192_square", 8192, 8192, 8192, dtype="fp16", scale="fp32"),
        # one request's next token: penalties and some biases (latency)
        _adjust("adjust_1", 1, 0, 600, 600, 20, "none"),
        # a batch of requests with histories of their own, into the sampler's 32 bits
        _adjust("adjust_64", 64, 0, 16, 4096, 8, "none", out="fp32"),
        # 64 sequences' five rows of a verify step: row i counts the i guesses before it
        _adjust("adjust_64_guesses", 64, 4, 64, 2048, 0, "none"),
        # structured output: a grammar's masks, most of them of few allowed tokens
        _adjust("adjust_64_masks", 64, 0, 1, 256, 0, "few", penalties=False),
        # long conversations, a small odd vocabulary, masks that ban few tokens
        _adjust("adjust_16_long", 16, 0, 20000, 120000, 300, "most", vocab=32003, dtype="fp32", out="fp32"),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    if rng.random() < 0.55:
        swiglu = rng.random() < 0.3
        m, k = _log(rng, 1, 8192), 16 * _log(rng, 4, 512)
        n = 32 * _log(rng, 1, 256) if swiglu else _log(rng, 16, 16384 if m > 100 else VOCAB)
        case = _product("", m, n, k, rng.random() < 0.5 and k <= 4096, swiglu, rng.choice(["bf16", "bf16", "fp16"]),
                        rng.choice(["bf16", "fp16", "fp32"]))
        if case["norm"]:
            case["dtype"] = "bf16"  # the framework's norms are bf16
    else:
        high = _log(rng, 4, 60000)
        vocab = _log(rng, 300, VOCAB)
        guesses = rng.choice([0, 0, 0, 2, 4, 8])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        seqs = _log(rng, 1, 256 // (1 + guesses))
        penalties = rng.random() < 0.8
        case = _adjust("", seqs, guesses, rng.randint(1, high), high, rng.choice([0, 0, 3, 40, 300]),
                       rng.choice(["none", "none", "few", "most"]), penalties, vocab, dtype, rng.choice([dtype, "fp32"]))
        case["bias"] = min(case["bias"], vocab // 2)
        if not penalties and not case["bias"] and case["masks"] == "none":
            case["masks"] = "most"
    del case["name"]
    return case


# ------------------------------------------------------------------------ lengths and work
def _lengths(case: dict) -> list[int]:
    """History lengths spread evenly over the case's range, in an order that the seed does not change."""
    lo, hi, n = case["len_lo"], case["len_hi"], case["seqs"]
    return [lo + (hi - lo) * ((7 * i) % n if n % 7 else i) // max(1, n - 1) for i in range(n)]


def work(case: dict) -> dict:
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        n_out = n // 2 if case["swiglu"] else n
        scale = DTYPES[case["scale"]].itemsize
        return {"bytes": 2 * m * k + n * k + scale * n + 2 * m * n_out + (2 * k if case["norm"] else 0), "flops": 2 * m * n * k}
    rows = case["seqs"] * (1 + case["guesses"])
    size = rows * case["vocab"]
    moved = size * (DTYPES[case["dtype"]].itemsize + DTYPES[case["out"]].itemsize) + 8 * rows * case["bias"]
    if case["penalties"]:
        moved += 4 * sum(_lengths(case)) + 4 * case["seqs"] * case["guesses"] + 12 * rows
    if case["masks"] != "none":
        moved += 4 * rows * ((case["vocab"] + 31) // 32)
    return {"bytes": moved, "flops": 4 * size}


# ------------------------------------------------------------------------ inputs
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return _prepare_product(case, g) if case["kind"] == "product" else _prepare_adjust(case, g)


def _prepare_product(case: dict, g: torch.Generator) -> dict:
    m, n, k = case["m"], case["n"], case["k"]
    dtype = DTYPES[case["dtype"]]
    # activations with outlier channels, as a transformer's are; rows of unlike size
    x = torch.randn((m, k), device="cuda", generator=g)
    channel = torch.rand(k, device="cuda", generator=g)
    x *= torch.where(channel > 0.99, 12.0, 0.5 + channel) * (0.25 + 2 * torch.rand((m, 1), device="cuda", generator=g))
    state = {"case": case, "x": x.to(dtype)}
    if case["norm"]:
        state["norm"] = (0.5 + torch.rand(k, device="cuda", generator=g)).to(dtype)
    state["w"] = torch.randn((n, k), device="cuda", generator=g).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
    state["w_scale"] = ((0.5 + torch.rand(n, device="cuda", generator=g)) / (36 * math.sqrt(k))).to(DTYPES[case["scale"]])
    return state


def _prepare_adjust(case: dict, g: torch.Generator) -> dict:
    seqs, vocab, guesses = case["seqs"], case["vocab"], case["guesses"]
    rows = seqs * (1 + guesses)
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=g)
    logits = 2.0 * torch.randn((rows, vocab), device="cuda", generator=g)
    likely = (uniform(rows, 40) * vocab).long().clamp_(max=vocab - 1)
    logits.scatter_add_(1, likely, 4.0 + 8.0 * uniform(rows, 40))
    state = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]),
             "out": torch.empty((rows, vocab), device="cuda", dtype=DTYPES[case["out"]])}
    # which sequence a row belongs to, and how many of its guesses come before the row
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    state["row_seq"] = state["row_guesses"] = state["guesses"] = None
    if guesses:
        state["row_seq"], state["row_guesses"] = row // (1 + guesses), row % (1 + guesses)
    if case["penalties"]:
        # text repeats itself: few tokens make up most of a history
        token = lambda *shape: (uniform(*shape).pow(4) * vocab).int().clamp_(max=vocab - 1)
        lens = _lengths(case)
        state["history"] = token(seqs, max(lens) + 8)
        state["history_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        state["prompt_len"] = (state["history_len"] * uniform(seqs)).int()
        if guesses:
            state["guesses"] = token(seqs, guesses)
        state["repetition"] = 1.0 + 0.4 * uniform(rows)
        state["presence"], state["frequency"] = 1.5 * uniform(rows) - 0.25, 0.5 * uniform(rows)
    if case["bias"]:
        n = case["bias"]
        # a window of the vocabulary in steps, another one for each row: no token twice in a row
        first = (uniform(rows, 1) * vocab).long()
        step = max(1, vocab // (2 * n))
        state["bias_tokens"] = ((first + step * torch.arange(n, device="cuda")) % vocab).int().reshape(-1)
        state["bias_values"] = 10.0 * uniform(rows * n) - 5.0
        state["bias_start"] = n * torch.arange(rows + 1, device="cuda", dtype=torch.int32)
    state["mask"] = None
    if case["masks"] != "none":
        words = (vocab + 31) // 32
        share = uniform(rows, 1).pow(6) * 0.5 if case["masks"] == "few" else 1.0 - 0.1 * uniform(rows, 1)
        mask = torch.zeros((rows, words), device="cuda", dtype=torch.int32)
        for bit in range(32):
            mask |= (uniform(rows, words) < share).int() << bit
        state["mask"] = mask
    return state


# ------------------------------------------------------------------------ a pass
def run(state: dict):
    case = state["case"]
    if case["kind"] == "product":
        return _product_own(state) if own else _product_plain(state)
    return _adjust_own(state) if own else _adjust_plain(state)


def _product_own(s: dict):
    kernels, case = _kernels(), s["case"]
    if case["norm"]:
        codes, scales = kernels.rmsnorm_quantize(s["x"], s["norm"], EPS)
    else:
        codes, scales = kernels.quantize_rows(s["x"])
    epilogue = kernels.EPILOGUE_SWIGLU if case["swiglu"] else kernels.EPILOGUE_STORE
    return kernels.w8a8_gemm(codes, scales, s["w"], s["w_scale"], epilogue=epilogue)


def _adjust_own(s: dict):
    kernels, case = _kernels(), s["case"]
    penalties = bias = None
    if case["penalties"]:
        penalties = kernels.TokenPenalties(s["history"], s["history_len"], s["prompt_len"], s["repetition"], s["presence"],
                                           s["frequency"], drafts=s["guesses"], row_seq=s["row_seq"], row_drafts=s["row_guesses"])
    if case["bias"]:
        bias = kernels.TokenBias(s["bias_start"], s["bias_tokens"], s["bias_values"])
    return kernels.adjust_logits(s["logits"], penalties=penalties, bias=bias, allowed=s["mask"], out=s["out"])


def _product_plain(s: dict):
    case, x = s["case"], s["x"].float()
    if case["norm"]:  # the framework's: both factors' results rounded to bf16
        x = (x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)).to(torch.bfloat16).float()
        x = (x * s["norm"].float()).to(torch.bfloat16).float()
    top = x.abs().amax(1, keepdim=True).clamp(min=1e-8)
    scale = (top.double() / 127.0).float()
    # the quotient in 32 bits, through 64: next to a half it decides the code
    codes = (x.double() / scale.double()).float().round().clamp(-127, 127)
    y = codes @ s["w"].float().t() * scale * s["w_scale"].float()
    if case["swiglu"]:
        pairs = y.view(case["m"], -1, 2, 16)
        gate, up = pairs[:, :, 0], pairs[:, :, 1]
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(case["m"], -1)
    return y.to(torch.bfloat16)


def _adjust_plain(s: dict):
    case, x = s["case"], s["logits"].float()
    rows, vocab = x.shape
    if case["penalties"]:
        history, length = s["history"].long(), s["history_len"].long()[:, None]
        at = torch.arange(history.shape[1], device="cuda")
        output = (at >= s["prompt_len"].long()[:, None]) & (at < length)
        count = torch.zeros((case["seqs"], vocab), device="cuda")
        count.scatter_add_(1, history, output.float())
        seen = torch.zeros((case["seqs"], vocab), device="cuda")
        seen.scatter_add_(1, history, (at < length).float())
        if case["guesses"]:
            seq = s["row_seq"].long()
            before = torch.arange(case["guesses"], device="cuda") < s["row_guesses"].long()[:, None]
            more = torch.zeros((rows, vocab), device="cuda").scatter_add_(1, s["guesses"].long()[seq], before.float())
            count, seen = count[seq] + more, seen[seq] + more
        r = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if case["bias"]:
        x = x.scatter_add(1, s["bias_tokens"].long().view(rows, -1), s["bias_values"].view(rows, -1))
    if s["mask"] is not None:
        token = torch.arange(vocab, device="cuda")
        x = x.masked_fill(s["mask"][:, token // 32] >> (token % 32) & 1 == 0, -math.inf)
    s["out"].copy_(x)
    return s["out"]


# ------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return _product_exact(s) if case["kind"] == "product" else _adjust_exact(s)


def _product_exact(s: dict) -> torch.Tensor:
    case = s["case"]
    x = s["x"].double()
    if case["norm"]:
        mean = (x * x).sum(1) / case["k"]
        x = ((x / torch.sqrt(mean + EPS)[:, None]).to(torch.bfloat16).double() * s["norm"].double()).to(torch.bfloat16).double()
    scale = (x.abs().max(1).values.clamp(min=1e-8) / 127).float().double()[:, None]
    codes = torch.clamp(torch.round(x / scale), -127, 127)
    out = torch.empty((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    for at in range(0, case["n"], 8192):  # a piece of the weights in 64 bits at a time
        piece = s["w"][at : at + 8192].double() * s["w_scale"][at : at + 8192].double()[:, None]
        out[:, at : at + 8192] = (codes * scale) @ piece.t().contiguous()
    if not case["swiglu"]:
        return out
    column = torch.arange(case["n"] // 2, device="cuda")
    gate = out[:, column // 16 * 32 + column % 16]
    up = out[:, column // 16 * 32 + 16 + column % 16]
    return gate * torch.sigmoid(gate) * up


def _adjust_exact(s: dict) -> torch.Tensor:
    """Row by row on the host."""
    case = s["case"]
    host = {name: t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()
            for name, t in s.items() if isinstance(t, torch.Tensor) and name != "out"}
    x = host["logits"]
    rows, vocab = x.shape
    for r in range(rows):
        if case["penalties"]:
            b = int(host["row_seq"][r]) if case["guesses"] else r
            tokens = host["history"][b, : host["history_len"][b]]
            made = tokens[host["prompt_len"][b] :]
            if case["guesses"]:
                extra = host["guesses"][b, : host["row_guesses"][r]]
                tokens, made = np.concatenate([tokens, extra]), np.concatenate([made, extra])
            seen = np.unique(tokens)
            value = x[r, seen]
            x[r, seen] = np.where(value > 0, value / host["repetition"][r], value * host["repetition"][r])
            distinct, counts = np.unique(made, return_counts=True)
            x[r, distinct] -= host["presence"][r] + host["frequency"][r] * counts
        if case["bias"]:
            part = slice(host["bias_start"][r], host["bias_start"][r + 1])
            x[r, host["bias_tokens"][part]] += host["bias_values"][part]
        if case["masks"] != "none":
            bits = np.unpackbits(host["mask"][r].view(np.uint8), bitorder="little")[:vocab]
            x[r, bits == 0] = -np.inf
    return torch.from_numpy(x).cuda()
