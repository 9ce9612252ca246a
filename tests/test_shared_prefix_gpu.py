"""Attention of batches that share prefixes (``kernels.shared_prefix_attention``) against plain
attention in 64 bits, sequence by sequence.

Tolerance, per output element, with A = sum p |v| / sum p of its row: the output's rounding to
bf16 is at most half a step, 2^-8 relative.  Probabilities enter the second product rounded
to bf16 (2^-8 relative, bf16 pools) or, times the value scale, to fp16 (2^-11, int8 pools,
and 2^-25 absolute beside a largest of 0.5 or more: for the up to 2^13 keys here below
2^-12 of A): each changes the row by at most its share of A.  Scores are sums of 128 fp32
products, 128 * 2^-24 of sum |q k| * scale (about 11 here): below 2^-13.  So
|got - ref| <= 2^-8 |ref| + (1 + 2^-8) c A, with c = 2^-8 + 2^-12 for bf16 pools and
2^-11 + 2^-12 + 2^-12 = 2^-10 for int8 pools.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from nanoengine_amd import _native, kernels

HEAD = 128


class Batch:
    """A pool, block tables that share their groups' first blocks, and queries.

    ``groups``: per group (shared tokens, members), a member being (own tokens before its
    queries, queries); a member None is an idle slot."""

    def __init__(self, groups, q_heads=16, kv_heads=8, kv="bf16", block=16, seed=0, scale_dtype=torch.bfloat16, shuffle=True,
                 gap=0, prefix_len=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        members = [(i, m) for i, (_, ms) in enumerate(groups) for m in ms]
        n = len(members)
        place = rng.permutation(n) if shuffle else np.arange(n)
        ceil = lambda t: -(-t // block)
        need = sum(ceil(p) for p, _ in groups) + sum(ceil(p % block + m[0] + m[1]) + 1 for p, ms in groups for m in ms if m)
        self.num_blocks = need + 3
        self.block, self.kv, self.q_heads, self.kv_heads = block, kv, q_heads, kv_heads
        free = list(rng.permutation(self.num_blocks))
        shared = [[free.pop() for _ in range(p // block)] for p, _ in groups]  # whole blocks are shared
        self.ctx, self.q_len = np.zeros(n, np.int32), np.zeros(n, np.int32)
        tables = [[] for _ in range(n)]
        for at, (i, m) in zip(place, members):
            if m is None:
                continue
            p = groups[i][0] // block * block
            self.ctx[at], self.q_len[at] = p + m[0] + m[1], m[1]
            tables[at] = shared[i] + [free.pop() for _ in range(ceil(m[0] + m[1]))]
        width = max(1, max(len(t) for t in tables))
        self.tables = np.zeros((n, width), np.int32)
        for at, t in enumerate(tables):
            self.tables[at, : len(t)] = t
        self.q_start = (np.concatenate([[0], np.cumsum(self.q_len + gap)[:-1]]) + gap).astype(np.int32)
        self.rows = int((self.q_len + gap).sum()) + gap
        order, start = [], [0]
        at = 0
        for _, ms in groups:
            order += [int(place[at + j]) for j in range(len(ms))]
            at += len(ms)
            start.append(at)
        self.group_lists = [order[a:b] for a, b in zip(start, start[1:])]
        self.prefix = [p // block * block for p, _ in groups] if prefix_len is None else prefix_len
        slots = self.num_blocks * block + 1
        k, v = (torch.randn(slots, kv_heads, HEAD, generator=g) for _ in range(2))
        if kv == "int8":
            def quantize(x):
                s = (x.abs().amax(-1) / 127).to(scale_dtype)
                return torch.clamp((x / s.float()[..., None]).round(), -127, 127).to(torch.int8), s
            (self.k, self.ks), (self.v, self.vs) = quantize(k), quantize(v)
        else:
            self.k, self.v, self.ks, self.vs = k.to(torch.bfloat16), v.to(torch.bfloat16), None, None
        self.q = (1.5 * torch.randn(max(self.rows, 1), q_heads, HEAD, generator=g)).to(torch.bfloat16)

    def to_gpu(self):
        for name in ("k", "v", "ks", "vs", "q"):
            t = getattr(self, name)
            setattr(self, name, None if t is None else t.cuda())
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
        self.d = {name: dev(getattr(self, name)) for name in ("tables", "ctx", "q_start", "q_len")}
        self.groups = kernels.PrefixGroups.from_lists(self.group_lists, self.prefix, torch.device("cuda:0"))
        return self

    def plan(self, max_q=None, max_ctx=None, **kwargs):
        return kernels.shared_prefix_plan(self.d["tables"], self.block, self.d["ctx"], self.d["q_start"], self.d["q_len"], self.groups,
                                          self.q_heads, self.kv_heads, max_q or max(1, int(self.q_len.max())),
                                          max_ctx or max(1, int(self.ctx.max())), num_rows=self.q.shape[0],
                                          num_blocks=self.num_blocks, **kwargs)

    def run(self, plan=None, out=None, scale=None):
        return kernels.shared_prefix_attention(self.q, self.k, self.v, self.ks, self.vs, plan or self.plan(), softmax_scale=scale,
                                               out=out)

    def reference(self, scale=None, max_ctx=1 << 30):
        """(rows, outputs, A) in 64 bits on the CPU."""
        scale = 1 / math.sqrt(HEAD) if scale is None else scale
        rows, outs, means = [], [], []
        k, v, q = (getattr(self, x).double().cpu() for x in "kvq")
        if self.kv == "int8":
            k, v = k * self.ks.double().cpu()[..., None], v * self.vs.double().cpu()[..., None]
        for s, (ctx, ql, qs) in enumerate(zip(self.ctx.tolist(), self.q_len.tolist(), self.q_start.tolist())):
            if ql == 0 or ctx == 0:
                continue
            p = torch.arange(min(ctx, max_ctx))
            slot = torch.from_numpy(self.tables[s]).long()[p // self.block] * self.block + p % self.block
            kk, vv = (x[slot].repeat_interleave(self.q_heads // self.kv_heads, 1).permute(1, 0, 2) for x in (k, v))
            qq = q[qs : qs + ql].permute(1, 0, 2)
            score = qq @ kk.transpose(1, 2) * scale
            score = score.masked_fill(p[None, :] > (ctx - ql + torch.arange(ql))[:, None], -math.inf)
            prob = torch.softmax(score, -1)
            hidden = (score == -math.inf)
            prob = torch.where(hidden, 0.0, prob)
            clean = torch.nan_to_num(vv, 0.0, 0.0, 0.0)
            rows += range(qs, qs + ql)
            outs.append((prob @ clean).permute(1, 0, 2))
            means.append((prob @ clean.abs()).permute(1, 0, 2))
        if not rows:
            return rows, torch.zeros(0, self.q_heads, HEAD), torch.zeros(0, self.q_heads, HEAD)
        return rows, torch.cat(outs), torch.cat(means)

    def check(self, out, scale=None, max_ctx=1 << 30):
        rows, ref, mean = self.reference(scale, max_ctx)
        c = 2.0**-10 if self.kv == "int8" else 2.0**-8 + 2.0**-12
        got = out.double().cpu()[rows]
        excess = (got - ref).abs() - (2.0**-8 * ref.abs() + (1 + 2.0**-8) * c * mean + 1e-30)
        assert bool((excess <= 0).all()), f"worst excess {float(excess.max()):.3g}, worst error {float((got - ref).abs().max()):.3g}"


MEMBERS = [(0, 1), (5, 1), (16, 1), (40, 1), (130, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("prefix", [0, 16, 48, 128, 144, 544, 2000])
def test_one_group_of_single_queries(kv, prefix):
    b = Batch([(prefix, MEMBERS)], kv=kv, seed=prefix).to_gpu()
    plan = b.plan()
    b.check(b.run(plan))
    assert plan.error_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv,scale_dtype", [("bf16", None), ("int8", torch.bfloat16), ("int8", torch.float16)])
@pytest.mark.parametrize("heads", [(16, 8), (8, 8), (32, 8), (4, 1), (14, 2), (24, 3), (32, 4), (5, 5), (40, 10), (71, 1)])
def test_head_layouts(kv, scale_dtype, heads):
    b = Batch([(96, [(3, 2), (20, 1), (0, 3)]), (0, [(50, 1)])], *heads, kv=kv, seed=heads[0], scale_dtype=scale_dtype or torch.bfloat16)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("q", [1, 2, 5, 8, 9, 16, 17, 33, 70])
def test_query_lengths(kv, q):
    """Light items up to 32 rows per KV head, tiles beyond; row tiles of 64, 128 and 256."""
    b = Batch([(208, [(30, q), (1, max(1, q // 2)), (0, q), (300, 1)]), (64, [(10, q), (10, 1)])], kv=kv, seed=q)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("members", [2, 33, 64, 150])
def test_group_sizes(kv, members):
    b = Batch([(300, [(i % 50, 1 + i % 5) for i in range(members)])], kv=kv, seed=members)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("prefix,members,q", [(1024, 64, 1), (1040, 40, 3), (2000, 30, 1), (1500, 130, 2), (4112, 26, 5), (9000, 24, 2)])
def test_prefixes_read_once(kv, prefix, members, q):
    """Batches in which sharing pays: row tiles of 64, 128 and 256, stages that end inside a prefix's
    last keys, one part and many."""
    b = Batch([(prefix, [((7 * i) % 90, max(1, q - i % 3)) for i in range(members)])], kv=kv, seed=prefix).to_gpu()
    plan = b.plan()
    b.check(b.run(plan))
    assert plan.error_flag() == 0 and plan.shared_items() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (8, 2), (6, 1), (30, 5), (24, 12)])
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_prefixes_read_once_by_other_heads(kv, heads):
    groups = [(1600 + 16 * heads[1], [((5 * i) % 60, 1 + i % 4) for i in range(60)]), (2304, [(i, 2) for i in range(50)]), (48, [(3, 1), None])]
    b = Batch(groups, *heads, kv=kv, seed=heads[0]).to_gpu()
    plan = b.plan()
    b.check(b.run(plan))
    flag, shared = plan.error_flag(), plan.shared_items()
    assert flag == 0
    if heads[1] > 1:  # the keys of one head are too few for sharing to pay
        assert shared > 0


@pytest.mark.gpu
def test_short_prefixes_are_read_by_each():
    b = Batch([(64, [(9, 1), (20, 1)])]).to_gpu()
    assert b.plan().shared_items() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_prompts_on_a_prefix_read_once(kv):
    """Members of more than 32 rows per KV head among single queries: own keys in tiles."""
    b = Batch([(1536, [(i, 1) for i in range(50)] + [(3, 40), (0, 70), (200, 33)])], kv=kv, seed=21).to_gpu()
    plan = b.plan()
    b.check(b.run(plan))
    assert plan.shared_items() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("block", [16, 32, 48, 128])
def test_block_sizes(kv, block):
    b = Batch([(5 * block, [(7, 3), (block, 1), (2 * block - 1, 1)]), (block, [(0, 2), (9, 1)])], kv=kv, block=block, seed=block)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_many_groups_of_unlike_sizes(kv):
    rng = np.random.default_rng(3)
    groups = [(int(rng.integers(0, 1500)), [(int(rng.integers(0, 400)), int(rng.integers(1, 10))) for _ in range(int(rng.integers(1, 9)))])
              for _ in range(20)]
    b = Batch(groups, kv=kv, seed=4).to_gpu()
    plan = b.plan()
    b.check(b.run(plan))
    assert plan.error_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_long_prefix_and_long_own_contexts(kv):
    b = Batch([(7000, [(10, 1), (900, 1), (0, 5)]), (16, [(6000, 4), (3000, 1)])], kv=kv, seed=5)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_prompts_on_a_shared_prefix(kv):
    """Prefill: hundreds of queries per sequence over the shared keys and their own."""
    b = Batch([(512, [(0, 300), (0, 129), (77, 200)]), (0, [(0, 65)])], kv=kv, seed=6)
    b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_idle_slots_and_rows_of_no_sequence(kv):
    """Idle members anywhere in a group (the first included), groups that shrink to one or none, and
    rows between the sequences that stay as they were."""
    b = Batch([(160, [None, (4, 2), None, (9, 1)]), (160, [None, (3, 1)]), (64, [None, None]), (0, [(8, 3)])], kv=kv, seed=7, gap=2).to_gpu()
    out = torch.full_like(b.q, 7.0)
    b.run(out=out)
    b.check(out)
    rows = set(b.reference()[0])
    rest = [i for i in range(b.rows) if i not in rows]
    assert rest and (out[rest] == 7).all()


@pytest.mark.gpu
def test_a_wholly_idle_batch_and_an_empty_one():
    b = Batch([(32, [None, None])], gap=1).to_gpu()
    out = torch.full_like(b.q, 3.0)
    b.run(out=out)
    assert (out == 3).all()
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    plan = kernels.shared_prefix_plan(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), 16, empty, empty, empty,
                                      kernels.PrefixGroups.from_lists([], [], torch.device("cuda:0")), 16, 8, 1, 1)
    q = torch.zeros(0, 16, HEAD, dtype=torch.bfloat16, device="cuda")
    assert kernels.shared_prefix_attention(q, b.k, b.v, None, None, plan).shape == (0, 16, HEAD)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_prefix_lengths_that_the_lengths_cut(kv):
    """A stated prefix off the 16-key grid, or reaching into a member's queries, is cut to what holds."""
    groups = [(320, [(0, 4), (50, 1)]), (320, [(2, 1), (3, 1)])]
    for stated in ([320, 320], [319, 17], [500, 330], [0, 1], [321, 336]):
        b = Batch(groups, kv=kv, seed=8, prefix_len=stated).to_gpu()
        # (members share 320 tokens: more is stated only where no more can be used)
        b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("scale", [0.0, 0.01, 1.0])
def test_softmax_scales(kv, scale):
    """Flat rows, and rows where one key takes all (scores up to ~100: 128 2^-24 sum |q k| is 1e-3)."""
    b = Batch([(256, [(30, 2), (64, 1)])], kv=kv, seed=9).to_gpu()
    if scale < 1:
        b.check(b.run(scale=scale), scale)
    else:
        rows, ref, mean = b.reference(scale)
        got = b.run(scale=scale).double().cpu()[rows]
        # where the one key holds a 0, fp16's absolute step is all that is left: a probability times
        # the value scale is off by up to 2^-25 beside a largest scale of 0.5 or more and a row sum of
        # 1 or more, so each of the keys adds at most 2^-25 * 2 * (127 * its scale) = 2^-24 max |v|
        step = int(b.ctx.max()) * 2.0**-24 * float((b.v.float().abs() * b.vs.float()[..., None]).max()) if kv == "int8" else 0.0
        excess = (got - ref).abs() - (2.0**-8 * ref.abs() + (2.0**-7 + 2e-3) * mean + step)
        assert bool((excess <= 0).all()), f"worst excess {float(excess.max()):.3g}, step {step:.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_scores_far_from_zero(kv):
    """A common offset of all scores (here about +-900 in log2) leaves the softmax as it is."""
    b = Batch([(256, [(30, 2), (64, 1)])], kv=kv, seed=10)
    b.q[:, :, 0] = 120.0
    kk = b.k.float() * b.ks.float()[..., None] if kv == "int8" else b.k.float()
    for sign in (1.0, -1.0):
        kk[:, :, 0] = sign * 60.0
        if kv == "int8":
            b.ks = (kk.abs().amax(-1) / 127).to(torch.bfloat16)
            b.k = torch.clamp((kk / b.ks.float()[..., None]).round(), -127, 127).to(torch.int8)
        else:
            b.k = kk.to(torch.bfloat16)
        b.to_gpu()
        rows, ref, mean = b.reference()
        got = b.run().double().cpu()[rows]
        # sum |q k| * scale is about 650: the scores' rounding 128 * 2^-24 * 650 = 5e-3 at most
        c = (2.0**-10 if kv == "int8" else 2.0**-8 + 2.0**-12) + 1e-2
        excess = (got - ref).abs() - (2.0**-8 * ref.abs() + (1 + 2.0**-8) * c * mean)
        assert bool((excess <= 0).all()), f"worst excess {float(excess.max()):.3g}"
        b.k, b.ks, b.q, b.v, b.vs = (None if t is None else t.cpu() for t in (b.k, b.ks, b.q, b.v, b.vs))


@pytest.mark.gpu
def test_small_and_unlike_value_scales():
    """Values of 1e-4 and of 1e4 in one int8 pool keep their relative precision."""
    for factor in (1e-5, 1e4, None):
        b = Batch([(400, [(30, 2), (164, 1), (5, 20)])], kv="int8", seed=11)
        if factor is None:  # each head of its own size
            b.vs = (b.vs.float() * (10.0 ** torch.linspace(-6, 4, 8))).to(torch.bfloat16)
        else:
            b.vs = (b.vs.float() * factor).to(torch.bfloat16)
        b.to_gpu().check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("q", [4, 24])
def test_hidden_keys_never_reach_a_row(kv, bad, q):
    """Keys and values that hold no numbers: past the end of a context, and at a later guess's
    position for the rows before it."""
    b = Batch([(128, [(20, q), (37, q)])], kv=kv, seed=12)
    cache_k, cache_v = (b.ks, b.vs) if kv == "int8" else (b.k, b.v)
    touched = []
    for s in range(2):
        ctx = int(b.ctx[s])
        last = b.tables[s][(ctx - 1) // 16] * 16
        for at in range((ctx - 1) % 16 + 1, 16):  # stale slots behind the context
            cache_k[last + at] = bad
            cache_v[last + at] = bad
        touched.append(int(last + (ctx - 1) % 16))
    b.to_gpu()
    b.check(b.run())
    cache_k, cache_v = (b.ks, b.vs) if kv == "int8" else (b.k, b.v)
    clean = b.run()
    for slot in touched:  # the last guess's own key: seen by its own row alone
        cache_v[slot] = bad
        cache_k[slot] = bad
    got = b.run()
    for s in range(2):
        a, n = int(b.q_start[s]), int(b.q_len[s])
        # the other rows go another way through the values: equal up to twice the tolerance
        assert torch.isfinite(got[a : a + n - 1]).all()
        assert float((got[a : a + n - 1].float() - clean[a : a + n - 1].float()).abs().max()) < 0.05
        assert not torch.isfinite(got[a + n - 1].float()).all()


@pytest.mark.gpu
def test_more_queries_than_context():
    """Queries before position 0 see nothing: their rows are zero."""
    b = Batch([(0, [(0, 6), (3, 2)])], seed=13).to_gpu()
    b.ctx[:] = np.where(b.q_len == 6, 2, b.ctx)
    b.d["ctx"].copy_(torch.from_numpy(b.ctx))
    out = b.run()
    s = int(np.argmax(b.q_len == 6))
    a = int(b.q_start[s])
    assert (out[a : a + 4] == 0).all() and torch.isfinite(out.float()).all()
    assert float(out[a + 4].float().abs().max()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_strided_queries_and_outputs(kv):
    b = Batch([(112, [(9, 3), (40, 2)])], kv=kv, seed=14).to_gpu()
    packed = torch.full((b.rows, 3, 16, HEAD), -2.0, dtype=torch.bfloat16, device="cuda")
    packed[:, 1] = b.q
    flat = b.q
    want = b.run()
    b.q = packed[:, 1]
    store = torch.full((b.rows, 20, HEAD + 8), -2.0, dtype=torch.bfloat16, device="cuda")
    out = store[:, 2:18, :HEAD]
    b.run(out=out)
    assert torch.equal(out, want) and (store[:, :2] == -2).all() and (store[:, 18:] == -2).all() and (store[..., HEAD:] == -2).all()
    b.q = flat


@pytest.mark.gpu
def test_bounds_on_lengths_flag_and_hold():
    b = Batch([(160, [(40, 2), (9, 1)])], seed=15).to_gpu()
    plan = b.plan(max_ctx=170)  # one context is longer: keys past 170 are dropped, its queries keep their positions
    b.check(b.run(plan), max_ctx=170)
    assert plan.error_flag() & 1
    plan = b.plan(max_q=1)  # a sequence of more queries is not computed
    out = torch.full_like(b.q, 5.0)
    b.run(plan, out=out)
    s = int(np.argmax(b.q_len == 2))
    a = int(b.q_start[s])
    assert plan.error_flag() & 2 and (out[a : a + 2] == 5).all()


@pytest.mark.gpu
def test_bad_groups_and_tables_are_flagged_and_stay_inside():
    b = Batch([(160, [(40, 2), (9, 1), (3, 1)]), (32, [(4, 1)])], seed=16).to_gpu()
    good = b.groups
    lists = [(good.seqs.clone().fill_(0), good.start), (good.seqs + 1, good.start), (good.seqs - 1, good.start),
             (good.seqs, good.start + 1), (good.seqs, good.start.flip(0).contiguous()), (good.seqs, good.start * 1000)]
    for seqs, start in lists:
        b.groups = kernels.PrefixGroups(seqs.contiguous(), start.contiguous(), good.prefix_len, good.max_prefix_len)
        plan = b.plan()
        out = torch.full_like(b.q, 9.0)
        b.run(plan, out=out)
        assert plan.error_flag() & 4
        assert torch.isfinite(out.float()).all()
    b.groups = good
    broken = b.d["tables"].clone()
    broken[0, 0], broken[1, 1] = -5, b.num_blocks + 100
    b.d["tables"] = broken
    plan = b.plan()
    b.run(plan)
    assert plan.error_flag() & 8
    b.d["q_start"] = torch.full_like(b.d["q_start"], b.rows)
    plan = b.plan()
    out = torch.full_like(b.q, 9.0)
    b.run(plan, out=out)
    assert plan.error_flag() & 2 and (out == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_a_captured_step_follows_its_lengths_and_groups(kv):
    """One graph of a plan and two layers, replayed over batches of other lengths, groups and contents."""
    dev = torch.device("cuda:0")
    first = Batch([(320, [(40, 3), (9, 3), (100, 2)]), (64, [(4, 1), None])], kv=kv, seed=17).to_gpu()
    n, width, rows = 5, 40, 20
    buf = {"tables": torch.zeros(n, width, dtype=torch.int32, device=dev), "ctx": torch.zeros(n, dtype=torch.int32, device=dev),
           "q_start": torch.zeros(n, dtype=torch.int32, device=dev), "q_len": torch.zeros(n, dtype=torch.int32, device=dev)}
    groups = kernels.PrefixGroups(torch.zeros(n, dtype=torch.int32, device=dev), torch.zeros(n + 1, dtype=torch.int32, device=dev),
                                  torch.zeros(n, dtype=torch.int32, device=dev), 512)
    slots = 60 * 16 + 1
    k, v = torch.zeros(slots, 8, HEAD, dtype=first.k.dtype, device=dev), torch.zeros(slots, 8, HEAD, dtype=first.k.dtype, device=dev)
    ks = vs = None
    if kv == "int8":
        ks, vs = torch.zeros(slots, 8, dtype=torch.bfloat16, device=dev), torch.zeros(slots, 8, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(2, rows, 16, HEAD, dtype=torch.bfloat16, device=dev)
    out = torch.zeros_like(q)

    def step():
        plan = kernels.shared_prefix_plan(buf["tables"], 16, buf["ctx"], buf["q_start"], buf["q_len"], groups, 16, 8, 4, 600,
                                          num_rows=rows, num_blocks=60)
        for i in range(2):
            kernels.shared_prefix_attention(q[i], k, v, ks, vs, plan, out=out[i])

    def fill(b):
        for name, t in buf.items():
            t.zero_()
            x = b.d[name]
            t[: x.shape[0]][..., : x.shape[-1]].copy_(x) if x.dim() == 2 else t[: x.shape[0]].copy_(x)
        m, g = b.groups.seqs.shape[0], b.groups.prefix_len.shape[0]
        rest = torch.arange(m, n, dtype=torch.int32, device=dev)
        groups.seqs.copy_(torch.cat([b.groups.seqs, rest]))  # slots of no sequence: empty groups' entries at the end
        groups.start.fill_(n)
        groups.start[: g + 1].copy_(b.groups.start)
        groups.prefix_len.zero_()
        groups.prefix_len[:g].copy_(b.groups.prefix_len)
        for name, t in (("k", k), ("v", v), ("ks", ks), ("vs", vs)):
            if t is not None:
                t.zero_()
                t[: getattr(b, name).shape[0]].copy_(getattr(b, name))
        q[0, : b.q.shape[0]].copy_(b.q)
        q[1, : b.q.shape[0]].copy_(b.q.flip(0))

    fill(first)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        shapes = [[(320, [(40, 3), (9, 3), (100, 2)]), (64, [(4, 1), None])], [(16, [(0, 1), (1, 1)])],
                  [(160, [None, (5, 4)]), (176, [(2, 1), (40, 2)])], [(480, [(0, 2), (1, 1), (30, 4), (9, 1), (60, 1)])]]
        b = Batch(shapes[seed], kv=kv, seed=30 + seed).to_gpu()
        fill(b)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        b.check(out[0, : b.q.shape[0]])
        eager = out.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    batches = [Batch([(640, [(i % 40, 3) for i in range(24)])], kv="int8", seed=40 + i).to_gpu() for i in range(2)]
    want = [b.run() for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s, b in zip(streams, batches):
            with torch.cuda.stream(s):
                got.append(b.run())
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


@pytest.mark.gpu
def test_slots_past_4_gib():
    """A pool whose last blocks lie beyond 32-bit byte offsets."""
    b = Batch([(64, [(9, 1), (20, 2)])], seed=18).to_gpu()
    want = b.run()
    extra = (5 << 30) // (16 * 8 * HEAD * 2)
    slots = (extra + b.num_blocks) * 16 + 1
    k, v = torch.empty(slots, 8, HEAD, dtype=torch.bfloat16, device="cuda"), torch.empty(slots, 8, HEAD, dtype=torch.bfloat16, device="cuda")
    k[extra * 16 :].copy_(b.k)
    v[extra * 16 :].copy_(b.v)
    b.k, b.v, b.num_blocks = k, v, extra + b.num_blocks
    b.d["tables"] = b.d["tables"] + extra
    plan = b.plan()
    assert torch.equal(b.run(plan), want) and plan.error_flag() == 0


# -------------------------------------------------------------------- refusals
def test_host_checks_refuse_before_a_launch():
    lib = _native.load()
    p, ws = ctypes.c_void_p(256), ctypes.c_size_t(1 << 40)
    size = lib.ne_shared_prefix_workspace_size
    assert size(4, 1, 16, 8, 5, 1000, 512) > 0
    for bad in [(0, 0, 16, 8, 1, 1, 0), (4, 5, 16, 8, 1, 1, 0), (4, 1, 16, 7, 1, 1, 0), (4, 1, 16, 8, 0, 1, 0), (4, 1, 16, 8, 1, 0, 0),
                (1025, 1, 16, 8, 1, 1, 0), (4, 1, 16, 8, 1, 100, -1), (4, 1, 0, 0, 1, 1, 0)]:
        assert size(*bad) == 0, bad

    def plan(seqs=4, groups=1, hq=16, hkv=8, q=5, ctx=1000, prefix=512, bs=16, blocks=100, ws_ptr=p, nbytes=ws, lens=p, rows=20):
        return lib.ne_shared_prefix_plan(lens, p, p, rows, p, p, p, seqs, groups, hq, hkv, q, ctx, prefix, 64, bs, blocks, ws_ptr, nbytes, None)

    assert plan(seqs=0) == 0  # nothing to do
    assert plan(seqs=2000) == -2 and plan(bs=8) == -2 and plan(bs=24) == -2
    for kwargs in (dict(seqs=-1), dict(groups=5), dict(hkv=7), dict(q=0), dict(ctx=0), dict(prefix=-1), dict(blocks=0),
                   dict(ws_ptr=None), dict(ws_ptr=ctypes.c_void_p(8)), dict(lens=None), dict(rows=-1)):
        assert plan(**kwargs) == -1, kwargs
    assert plan(nbytes=ctypes.c_size_t(1000)) == -4 and b"needed" in lib.ne_last_error()

    def attend(q=p, ks=p, kv=3, sdt=0, dim=128, stride=2048, ws_ptr=p, scale=0.1):
        return lib.ne_shared_prefix_attention(q, stride, 128, p, p, ks, p, kv, sdt, p, 64, 16, 100, 4, 1, 16, 8, dim, 5, 1000, 512, scale, p,
                                              2048, 128, ws_ptr, ws, None)

    assert attend(dim=64) == -2
    for kwargs in (dict(q=None), dict(ks=None), dict(kv=1), dict(sdt=2), dict(stride=2047), dict(q=ctypes.c_void_p(264)), dict(ws_ptr=None),
                   dict(scale=math.nan)):
        assert attend(**kwargs) == -1, kwargs


def test_groups_from_lists_are_checked():
    cpu = torch.device("cpu")
    g = kernels.PrefixGroups.from_lists([[2, 0], [1]], [32, 0], cpu)
    assert g.seqs.tolist() == [2, 0, 1] and g.start.tolist() == [0, 2, 3] and g.prefix_len.tolist() == [32, 0] and g.max_prefix_len == 32
    for groups, lens in (([[0], [0]], [1, 1]), ([[0, 2]], [1]), ([[0]], [])):
        with pytest.raises(ValueError):
            kernels.PrefixGroups.from_lists(groups, lens, cpu)


@pytest.mark.gpu
def test_refusals_of_the_tensor_calls():
    b = Batch([(32, [(4, 1), (5, 1)])]).to_gpu()
    plan = b.plan()
    call = lambda **kw: kernels.shared_prefix_attention(**(dict(q=b.q, k_cache=b.k, v_cache=b.v, k_scale=None, v_scale=None, plan=plan) | kw))
    for kw in (dict(q=b.q.float()), dict(q=b.q[:, :8]), dict(k_cache=b.k[:, :4], v_cache=b.v[:, :4]), dict(k_cache=b.k.half(), v_cache=b.v.half()),
               dict(k_cache=b.k.to(torch.int8), v_cache=b.v.to(torch.int8)), dict(out=torch.empty_like(b.q[:1])), dict(q=b.q[:1])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(RuntimeError):
        call(q=b.q.cpu())
    with pytest.raises(ValueError):
        b.plan(workspace=torch.empty(100, device="cuda"))
    with pytest.raises(RuntimeError, match="NE_EWORKSPACE"):
        b.plan(workspace=torch.empty(512, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        b.d["ctx"] = b.d["ctx"].long()
        b.plan()
