"""Copying KV blocks and forking sequences: the pairs' checks and the allocators' fork on the
CPU, the copies on the GPU (bytes, so exact)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nanoengine_amd import _native, kernels
from nanoengine_amd.interface import GenerationRequest, SamplingParams
from nanoengine_amd.memory import KVCachePool, OutOfKVMemoryError, PagedSlotAllocator, PrefixCachingSlotAllocator
from nanoengine_amd.sequence_state import Sequence


def sequence(rid: str, tokens: list[int]) -> Sequence:
    return Sequence.from_request(GenerationRequest(rid, tokens, SamplingParams(max_new_tokens=64)))


# ----------------------------------------------------------------------- pairs
@pytest.mark.parametrize("src,dst,word", [([0], [8], b"block 0 -> 8"), ([-1], [1], b"block -1"), ([8], [1], b"block 8"),
                                          ([0, 1], [5, 5], b"twice"), ([0, 5], [5, 6], b"another copy's source"),
                                          ([2, 0], [2, 2], b"twice")])
def test_bad_pairs_are_refused_before_a_launch(src, dst, word):
    lib = _native.load()
    array = lambda kind, values: (kind * len(values))(*values)
    rc = lib.ne_kv_copy_blocks(array(ctypes.c_void_p, [4096]), array(ctypes.c_int64, [512]), 1, 8,
                               array(ctypes.c_int32, src), array(ctypes.c_int32, dst), len(src), None)
    assert rc == -1 and word in lib.ne_last_error()


def test_bad_buffers_and_sizes_are_refused():
    lib = _native.load()
    one = (ctypes.c_int32 * 1)(0)
    call = lambda buffers, block, n, blocks, pairs: lib.ne_kv_copy_blocks(
        (ctypes.c_void_p * 1)(buffers), (ctypes.c_int64 * 1)(block), n, blocks, one, one, pairs, None)
    assert call(None, 512, 1, 8, 1) == -1 and b"null" in lib.ne_last_error()
    assert call(4096, 0, 1, 8, 1) == -1 and b"bad block" in lib.ne_last_error()
    assert call(4096, 1 << 31, 1, 8, 1) == -1
    assert call(4096, 512, -1, 8, 1) == -1 and call(4096, 512, 1, 8, -1) == -1 and call(4096, 512, 1, -1, 1) == -1
    assert call(4096, 512, 0, 8, 1) == 0 and call(4096, 512, 1, 8, 0) == 0  # nothing to do
    assert lib.ne_kv_copy_blocks(None, None, 1, 8, one, one, 1, None) == -1


def test_cpu_buffers_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.copy_kv_blocks([torch.zeros(65, 2)], 16, [0], [1])
    with pytest.raises(ValueError):
        kernels.copy_kv_blocks([], 16, [0], [1])
    with pytest.raises(ValueError):
        kernels.copy_kv_blocks([torch.zeros(65, 2)], 16, [0, 1], [1])


# ------------------------------------------------------------------------ fork
def test_paged_fork_copies_every_block():
    a = PagedSlotAllocator(8, 16, torch.device("cpu"))
    a.reserve("p", 40)
    src, dst = a.fork("p", "c", 33)
    assert src == a.block_table("p") and dst == a.block_table("c") and not set(src) & set(dst)
    src, dst = a.fork("p", "d", 16)
    assert len(dst) == 1 and src == a.block_table("p")[:1]
    a.free("p")
    a.free("c")
    a.free("d")
    assert a.num_free_blocks == 8


def test_prefix_caching_fork_shares_full_blocks():
    a = PrefixCachingSlotAllocator(8, 16, torch.device("cpu"))
    p = sequence("p", list(range(40)))
    a.reserve(p, 40)
    p.num_cached_tokens = 40
    a.on_tokens_cached(p)
    src, dst = a.fork(p, "c", 40)
    assert a.block_table("c")[:2] == a.block_table(p)[:2] and a.block_table("c")[2] == dst[0] != src[0]
    assert a.first_writable_position(p) == a.first_writable_position("c") == 32
    assert all(a.pool.reference_count(b) == 2 for b in a.block_table(p)[:2])
    assert a.pool.reference_count(src[0]) == a.pool.reference_count(dst[0]) == 1
    # at a block's end nothing is copied
    assert a.fork(p, "d", 32) == ([], []) and a.block_table("d") == a.block_table(p)[:2]
    a.free(p)
    assert [a.pool.reference_count(b) for b in a.block_table("c")] == [2, 2, 1]
    a.free("c")
    a.free("d")
    assert a.num_free_blocks == 8


def test_forked_blocks_of_unregistered_tokens_are_not_written_either():
    a = PrefixCachingSlotAllocator(8, 16, torch.device("cpu"))
    p = sequence("p", list(range(50)))
    a.reserve(p, 50)  # cached but not yet registered
    assert a.first_writable_position(p) == 0
    a.fork(p, "c", 50)
    assert a.first_writable_position(p) == 48 and a.first_writable_position("c") == 48
    a.free("c")
    a.free(p)
    again = sequence("p", [1, 2])
    a.reserve(again, 2)
    assert a.first_writable_position(again) == 0  # a freed request leaves nothing behind


def test_a_child_registers_its_own_continuation():
    a = PrefixCachingSlotAllocator(12, 16, torch.device("cpu"))
    p = sequence("p", list(range(36)))
    a.reserve(p, 36)
    p.num_cached_tokens = 36
    a.on_tokens_cached(p)
    c = sequence("c", list(range(36)) + [99] * 12)
    a.fork(p, c, 36)
    a.reserve(c, 48)
    c.num_cached_tokens = 48
    a.on_tokens_cached(c)
    probe = sequence("probe", list(range(36)) + [99] * 12 + [5])
    assert a.find_cached_blocks(probe) == a.block_table(c)[:3]


def test_fork_refusals():
    for kind in (PagedSlotAllocator, PrefixCachingSlotAllocator):
        a = kind(3, 16, torch.device("cpu"))
        a.reserve("p", 40)
        with pytest.raises(OutOfKVMemoryError):
            a.fork("p", "c", 40)
        assert a.block_table("c") == [] and a.num_free_blocks == 0  # nothing taken
        with pytest.raises(ValueError, match="no blocks"):
            a.fork("q", "c", 1)
        with pytest.raises(ValueError, match="already"):
            a.fork("p", "p", 1)
        with pytest.raises(ValueError, match="holds no 49"):
            a.fork("p", "c", 49)
        with pytest.raises(ValueError):
            a.fork("p", "c", -1)


# ---------------------------------------------------------------------- copies
def reference(buffers, block_size, src, dst):
    out = [b.clone() for b in buffers]
    for s, d in zip(src, dst):
        for new, old in zip(out, buffers):
            new[d * block_size : (d + 1) * block_size] = old[s * block_size : (s + 1) * block_size]
    return out


def fill(pool, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for b in pool.buffers:
        b.view(torch.uint8).random_(0, 256, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("layers,heads,block", [(1, 8, 16), (3, 1, 16), (2, 3, 32), (28, 8, 16), (40, 2, 48)])
def test_copies_every_layer(int8, layers, heads, block):
    pool = KVCachePool(layers, heads, 128, 21 * block, torch.device("cuda:0"), torch.bfloat16, int8, block)
    fill(pool, layers)
    for src, dst in [([], []), ([3], [0]), ([20, 20, 4], [1, 2, 19]), ([5, 6], [5, 7]), (list(range(10)), list(range(10, 20)))]:
        want = reference(pool.buffers, block, src, dst)
        pool.copy_blocks(src, dst)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool.buffers, want))


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [223, 224, 225, 700])
def test_many_pairs_take_several_launches(pairs):
    pool = KVCachePool(2, 2, 128, 1500 * 16, torch.device("cuda:0"), torch.bfloat16, True, 16)
    fill(pool, pairs)
    order = torch.randperm(1500, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = order[:pairs], order[pairs : 2 * pairs]
    want = reference(pool.buffers, 16, src, dst)
    pool.copy_blocks(src, dst)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool.buffers, want))


@pytest.mark.gpu
@pytest.mark.parametrize("width,dtype,block,offset", [(5, torch.int8, 3, 0), (1, torch.bfloat16, 1, 1), (7, torch.float32, 2, 1),
                                                      (24, torch.int8, 4, 8)])
def test_blocks_off_the_vector_grid(width, dtype, block, offset):
    flat = torch.randint(-100, 100, (97 * width + offset,), device="cuda").to(dtype)
    buffer = flat[offset:].view(97, width)
    rest = flat[:offset].clone()
    want = reference([buffer], block, [0, 5], [7, 8])
    kernels.copy_kv_blocks([buffer], block, [0, 5], [7, 8])
    assert torch.equal(buffer, want[0]) and torch.equal(flat[:offset], rest)


@pytest.mark.gpu
def test_blocks_past_4_gib():
    slots = (5 << 30) // (8 * 128 * 2)
    buffer = torch.zeros(slots + 1, 8, 128, dtype=torch.bfloat16, device="cuda")
    last = slots // 16 - 1
    buffer[last * 16 : last * 16 + 16] = 3.0
    buffer[:16] = 2.0
    kernels.copy_kv_blocks([buffer], 16, [last, 0], [1, last - 1])
    assert (buffer[16:32] == 3).all() and (buffer[(last - 1) * 16 : last * 16] == 2).all()
    assert (buffer[32 : (last - 1) * 16] == 0).all()


@pytest.mark.gpu
def test_a_captured_copy_replays_its_pairs():
    pool = KVCachePool(4, 8, 128, 10 * 16, torch.device("cuda:0"), torch.bfloat16, True, 16)
    fill(pool, 1)
    graph = torch.cuda.CUDAGraph()
    pool.copy_blocks([], [])
    with torch.cuda.graph(graph):
        pool.copy_blocks([0, 1], [2, 3])
    for seed in range(3):
        fill(pool, 10 + seed)
        want = reference(pool.buffers, 16, [0, 1], [2, 3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool.buffers, want))


@pytest.mark.gpu
def test_refusals_of_the_tensor_call():
    pool = KVCachePool(2, 8, 128, 10 * 16, torch.device("cuda:0"), torch.bfloat16, False, 16)
    for src, dst in [([10], [0]), ([0], [-1]), ([0], [10])]:
        with pytest.raises(ValueError, match="outside"):
            pool.copy_blocks(src, dst)
    with pytest.raises(RuntimeError, match="twice"):
        pool.copy_blocks([0, 1], [2, 2])
    with pytest.raises(TypeError):
        pool.copy_blocks([0.5], [1])
    with pytest.raises(ValueError, match="contiguous"):
        kernels.copy_kv_blocks([pool.key_caches[0][:, :1]], 16, [0], [1])
    with pytest.raises(ValueError, match="same slots"):
        kernels.copy_kv_blocks([pool.key_caches[0], pool.key_caches[1][:100]], 16, [0], [1])
    with pytest.raises(ValueError):
        kernels.copy_kv_blocks(pool.buffers, 0, [0], [1])
