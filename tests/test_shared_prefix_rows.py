"""Shared-prefix attention of plans that were made before the rows of ``q`` are known."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from nanoengine_amd import _native, kernels
from test_shared_prefix_gpu import Batch


def plan_without_rows(b: Batch):
    return kernels.shared_prefix_plan(b.d["tables"], b.block, b.d["ctx"], b.d["q_start"], b.d["q_len"], b.groups, b.q_heads,
                                      b.kv_heads, int(b.q_len.max()), int(b.ctx.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("groups", [[(160, [(9, 3), (40, 5), (3, 2)]), (0, [(30, 2)])],  # light items
                                    [(96, [(9, 40), (40, 33)]), (0, [(30, 70)])],  # tiles of own keys
                                    [(2304, [((5 * i) % 60, 3) for i in range(70)])]])  # tiles of a group
def test_sequences_past_the_rows_of_q_are_left_out(kv, groups):
    b = Batch(groups, kv=kv, seed=50).to_gpu()
    want = b.run()
    plan = plan_without_rows(b)
    assert torch.equal(b.run(plan), want) and plan.error_flag() == 0  # all of them fit
    # q and out end one row into the sequence of the last rows
    last = int(np.argmax(b.q_start))
    rows = int(b.q_start[last]) + 1
    store_q, store_out = b.q, torch.full_like(b.q, 5.0)
    plan = plan_without_rows(b)
    kernels.shared_prefix_attention(store_q[:rows], b.k, b.v, b.ks, b.vs, plan, out=store_out[:rows])
    assert plan.error_flag() == 2
    assert torch.equal(store_out[: rows - 1], want[: rows - 1]) and (store_out[rows - 1 :] == 5).all()
    # a start behind everything, and one that 32 bits hold only just
    for start in (b.rows + 1000, 2**31 - 1 - int(b.q_len[last])):
        b.d["q_start"][last] = start
        plan = plan_without_rows(b)
        store_out.fill_(5.0)
        kernels.shared_prefix_attention(store_q, b.k, b.v, b.ks, b.vs, plan, out=store_out)
        assert plan.error_flag() == 2
        assert torch.equal(store_out[: rows - 1], want[: rows - 1]) and (store_out[rows - 1 :] == 5).all()


@pytest.mark.gpu
def test_a_batch_of_no_rows():
    b = Batch([(32, [None, None])]).to_gpu()
    none = b.q[:0]
    plan = kernels.shared_prefix_plan(b.d["tables"], b.block, b.d["ctx"], b.d["q_start"], b.d["q_len"], b.groups, 16, 8, 1, 1)
    assert kernels.shared_prefix_attention(none, b.k, b.v, None, None, plan).shape == (0, 16, 128)


def test_row_counts_are_checked_before_a_launch():
    lib = _native.load()
    p, ws = ctypes.c_void_p(256), ctypes.c_size_t(1 << 40)

    def attend(rows, q=p):
        return lib.ne_shared_prefix_attention_rows(q, 2048, 128, rows, p, p, p, p, 3, 0, p, 64, 16, 100, 4, 1, 16, 8, 128, 5, 1000, 512,
                                                   0.1, p, 2048, 128, p, ws, None)

    assert attend(-1) == -1 and b"row count" in lib.ne_last_error()
    assert attend(0) == 0 and attend(0, q=None) == 0  # nothing to compute
    assert attend(20, q=None) == -1 and b"null" in lib.ne_last_error()


@pytest.mark.gpu
def test_an_empty_batch_has_no_errors_and_no_items():
    """Its plan writes nothing, so what the workspace held before does not count."""
    dev = torch.device("cuda:0")
    empty = torch.zeros(0, dtype=torch.int32, device=dev)
    workspace = torch.full((4096,), 255, dtype=torch.uint8, device=dev)
    plan = kernels.shared_prefix_plan(torch.zeros(0, 1, dtype=torch.int32, device=dev), 16, empty, empty, empty,
                                      kernels.PrefixGroups.from_lists([], [], dev), 16, 8, 1, 1, workspace=workspace)
    assert plan.error_flag() == 0 and plan.shared_items() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("block_size", [0, -16, 8, 24])
def test_block_sizes_that_no_pool_has(block_size):
    b = Batch([(32, [(4, 1), (5, 1)])]).to_gpu()
    with pytest.raises(RuntimeError, match="block_size"):
        kernels.shared_prefix_plan(b.d["tables"], block_size, b.d["ctx"], b.d["q_start"], b.d["q_len"], b.groups, 16, 8, 1, 100)
