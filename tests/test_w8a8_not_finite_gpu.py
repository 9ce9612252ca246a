"""Rows that are not finite through the fused QKV product with 8-bit activations."""

from __future__ import annotations

import pytest
import torch

from nanoengine_amd import kernels
from test_w8a8_gpu import CACHES, qkv_case


@pytest.mark.gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("m", [5, 300])
def test_a_row_without_a_scale_spoils_its_own_vectors_alone(m, cache):
    """A row with a NaN or an infinity has the scale NaN (quantize_rows).  Its query and its vectors in a bf16
    cache are NaN.  An int8 cache has no NaN: the scale is that of a vector of zeros, 1e-8 / 127, so that what
    it stands for is at most 1e-8 (and half a step of the scale's type), by this product as by the row kernel
    after the plain one.  Every other row's bits are those of a batch without it."""
    hq, hkv, k = 4, 2, 256
    (codes, scales, w, w_scale), (q_norm, k_norm, eps, positions, rope, where), pool = qkv_case(m, hq, hkv, k, cache, seed=m)
    bad = torch.tensor([0, 3, m - 1], device="cuda")
    spoiled = scales.clone()
    spoiled[bad] = float("nan")
    queries, pools = [], []
    for s in (scales, spoiled):
        queries.append(torch.empty(m, hq, 128, device="cuda", dtype=torch.bfloat16))
        pools.append(pool())
        kernels.w8a8_qkv_norm_rope_kv(codes, s, w, w_scale, hq, hkv, q_norm, k_norm, eps, positions, rope, where, *pools[-1], queries[-1])
    two = pool()
    kernels.qk_norm_rope_kv_write(kernels.w8a8_gemm(codes, spoiled, w, w_scale), hq, hkv, q_norm, k_norm, eps, positions, rope, where, *two)
    kept = torch.ones(m, dtype=torch.bool, device="cuda")
    kept[bad] = False
    assert queries[1][bad].isnan().all() and torch.equal(queries[0][kept], queries[1][kept])
    other = torch.ones(m + 9, dtype=torch.bool, device="cuda")
    other[where[bad].long()] = False
    for clean, got in zip(pools[0], pools[1]):
        assert clean is got is None or torch.equal(clean[other], got[other])
    slots = where[bad].long()
    if cache[1] is None:
        assert pools[1][0][slots].isnan().all() and pools[1][1][slots].isnan().all()
        return
    for kernel in (pools[1], two):
        for codes_of, scale in ((kernel[0], kernel[2]), (kernel[1], kernel[3])):
            stands_for = codes_of[slots].double() * scale[slots].double()[..., None]
            assert float(stands_for.abs().max()) <= 1e-8 * (1 + 2.0**-8)
    assert torch.equal(pools[1][2][slots], two[2][slots]) and torch.equal(pools[1][3][slots], two[3][slots])
