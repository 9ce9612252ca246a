"""Rows quantised to int8 and W8A8 products against their definitions in 64 bits.

Codes and scales have to be equal.  A product's sum is exact; its fp32 value (one rounding), the two
scale factors (one each) and the rounding to bf16 give |y - y64| <= (2^-8 + 3 * 2^-24 * (1 + 2^-8)) |y64|,
taken as 2^-8 + 2^-22.  SwiGLU: gate g and up u are off by 3 * 2^-24 relative; silu(g) changes by
(1 + |g|) times g's relative error, exp's argument is rounded once (|g| 2^-24) and exp, the sum, the
quotient and the product add at most 2^-21: for |g| <= 60 at most 61 * 3 * 2^-24 + 60 * 2^-24 + 2^-21 +
3 * 2^-24 < 2^-15 relative, next to bf16's 2^-8.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from nanoengine_amd import _native, kernels
from nanoengine_amd._native import EPILOGUE_STORE, EPILOGUE_SWIGLU

STORE_REL = 2.0**-8 + 2.0**-22
SWIGLU_REL = 2.0**-8 + 2.0**-15
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rows_reference(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): the fp32 quotients correctly rounded, through 64 bits."""
    top = x.double().abs().amax(1).clamp(min=float(torch.tensor(1e-8)))
    scales = (top / 127).float()
    codes = (x.double() / scales.double()[:, None]).float().round().clamp(-127, 127)
    bad = ~torch.isfinite(x.float()).all(1)
    return codes.nan_to_num(0.0, 0.0, 0.0).masked_fill(bad[:, None], 0).to(torch.int8), scales.masked_fill(bad, float("nan"))


def check_rows(got, x) -> None:
    codes, scales = rows_reference(x)
    assert torch.equal(got[0], codes)
    assert torch.equal(got[1].nan_to_num(-1.0), scales.nan_to_num(-1.0))


def make(m, n, k, seed=0, scale="bf16"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-127, 128, (m, k), device="cuda", generator=g, dtype=torch.int32).to(torch.int8)
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int32).to(torch.int8)
    scales = 0.01 + 0.02 * torch.rand(m, device="cuda", generator=g)
    w_scale = ((0.5 + torch.rand(n, device="cuda", generator=g)) / (73 * k**0.5)).to(DTYPES[scale])
    return codes, scales, w, w_scale


def product(codes, scales, w, w_scale) -> torch.Tensor:
    y = codes.double() @ w.double().t().contiguous()
    return y * scales.double()[:, None] * w_scale.double()


def swiglu(y: torch.Tensor) -> torch.Tensor:
    gate, up = y.view(y.shape[0], -1, 2, 16).unbind(2)
    assert float(gate.abs().max()) <= 60
    return (gate * torch.sigmoid(gate) * up).reshape(y.shape[0], -1)


def check_product(got, codes, scales, w, w_scale, epilogue=EPILOGUE_STORE) -> None:
    want = product(codes, scales, w, w_scale)
    rel = STORE_REL
    if epilogue == EPILOGUE_SWIGLU:
        want, rel = swiglu(want), SWIGLU_REL
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    off = (got.double() - want).abs() - rel * want.abs()
    assert float(off.max()) <= 1e-38


# ------------------------------------------------------------------------- rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,k", [(1, 8), (3, 16), (5, 504), (4, 512), (7, 520), (9, 1024), (2, 2040), (6, 4096),
                                    (3, 4104), (2, 8192), (3, 16376), (2, 16392), (1, 131056), (1025, 128),
                                    (512, 2048), (513, 2048), (514, 1032), (30, 2056)])
def test_quantize_rows(rows, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * k)
    x = torch.randn(rows, k, device="cuda", generator=g) * (0.01 + 50 * torch.rand(rows, 1, device="cuda", generator=g))
    x = x.to(DTYPES[dtype])
    check_rows(kernels.quantize_rows(x), x)


@pytest.mark.gpu
def test_quantize_rows_ties_zeros_and_extremes():
    k = 256
    x = torch.zeros(7, k, device="cuda", dtype=torch.bfloat16)
    x[1, :] = torch.arange(k, device="cuda") * 0.5 - 63.5  # scale 0.5: quotients on and next to halves
    x[1, 0] = 63.5
    x[2, 3] = 1e-38  # far below the least scale
    x[3, 7] = torch.finfo(torch.bfloat16).max
    x[4, :] = -2.0**-126
    x[5, 11] = 127.0
    x[5, 12], x[5, 13], x[5, 14] = 0.5, 1.5, -2.5  # scale 1: ties to even
    x[6] = torch.randn(k, device="cuda")
    got = kernels.quantize_rows(x)
    check_rows(got, x)
    assert got[0][5, 12:15].tolist() == [0, 2, -2]


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("k", [64, 5000, 20000])
def test_rows_that_are_not_finite(k, value):
    x = torch.randn(3, k, device="cuda").bfloat16()
    x[1, k - 1] = value
    codes, scales = kernels.quantize_rows(x)
    check_rows((codes, scales), x)
    part = codes[:, : k // 16 * 16].contiguous()  # (products take a k of whole 16s)
    y = kernels.w8a8_gemm(part, scales, torch.ones_like(part[:1]).expand(16, -1).contiguous(), torch.ones(16, device="cuda"))
    assert y[1].isnan().all() and not y[0].isnan().any() and not y[2].isnan().any()


@pytest.mark.gpu
def test_quantize_rows_of_a_strided_view_into_given_outputs():
    big = torch.randn(9, 1024 + 64, device="cuda").bfloat16()
    x = big[:, 64:]
    codes = torch.full((11, 1024), 99, device="cuda", dtype=torch.int8)
    scales = torch.full((11,), 99.0, device="cuda")
    got = kernels.quantize_rows(x, codes=codes[1:10], scales=scales[1:10])
    check_rows(got, x)
    assert (codes[0] == 99).all() and (codes[10] == 99).all() and scales[0] == 99 and scales[10] == 99


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(1, 8), (5, 512), (3, 1024), (66, 1032), (7, 2048), (4, 4096)])
def test_norm_rows_are_the_norms_bits(rows, hidden):
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x = (3 * torch.randn(rows, hidden, device="cuda", generator=g)).bfloat16()
    delta = torch.randn(rows, hidden, device="cuda", generator=g).bfloat16()
    weight = (0.5 + torch.rand(hidden, device="cuda", generator=g)).bfloat16()
    check_rows(kernels.rmsnorm_quantize(x, weight, 1e-6), kernels.rmsnorm(x, weight, 1e-6))
    one, two = x.clone(), x.clone()
    got = kernels.add_rmsnorm_quantize(one, delta, weight, 1e-6)
    check_rows(got, kernels.add_rmsnorm(two, delta, weight, 1e-6))
    assert torch.equal(one, two)
    # and the norm's definition in 64 bits: two roundings to bf16 and half a step of the codes
    h = one.double()
    want = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * weight.double()
    s = got[1].double()[:, None]
    assert ((got[0].double() * s - want).abs() <= s * 0.5001 + want.abs() * (2 * 2.0**-8 + 2.0**-15)).all()


# ----------------------------------------------------------------------- products
SHAPES = [
    (1, 1, 16), (1, 15, 32), (1, 17, 48), (2, 4096, 1024), (15, 130, 112), (16, 541, 128), (17, 64, 1040), (33, 100, 2048),
    (64, 1024, 2048), (48, 33, 4112), (65, 64, 16), (65, 127, 80), (100, 541, 608), (127, 129, 64), (128, 128, 192),
    (200, 1000, 144), (129, 32003, 64), (64, 40000, 96), (3, 70000, 272), (300, 8192, 1024), (1000, 2048, 336), (2049, 4100, 80),
    (1111, 9001, 1024), (4096, 2304, 208), (9000, 9100, 80), (4100, 5003, 1040), (8192, 4096, 256), (2048, 16384, 400), (350, 64, 2064),
    (64, 151936, 64), (520, 4104, 144), (129, 4160, 2048),
]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k):
    data = make(m, n, k, seed=m + n + k, scale=["bf16", "fp16", "fp32"][(m + n) % 3])
    check_product(kernels.w8a8_gemm(*data), *data)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 32, 16), (1, 6144, 1024), (16, 96, 144), (31, 64, 1024), (64, 512, 272), (65, 32, 48),
                                   (150, 320, 64), (333, 6144, 1024), (700, 4096, 176), (2100, 5152, 336), (200, 192, 1040), (20, 6144, 528),
                                   (9000, 9120, 144), (4100, 8192, 1040), (40, 40000, 64), (257, 4128, 2064)])
def test_swiglu_product(m, n, k):
    data = make(m, n, k, seed=m + n + k)
    check_product(kernels.w8a8_gemm(*data, epilogue=EPILOGUE_SWIGLU), *data, epilogue=EPILOGUE_SWIGLU)


def test_every_kernel_serves_some_shape():
    if not _native.library_path().exists():
        pytest.skip("libnanoengine_hip.so is not built")
    lib = _native.load()
    assert {lib.ne_w8a8_kernel(m, n, k, EPILOGUE_STORE) for m, n, k in SHAPES} == {0, 1, 2, 3, 4}


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(5, 100, 64), (70, 250, 160), (300, 4096, 128), (2200, 4096, 64)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_product_strides_and_what_lies_beside_it(m, n, k, pad):
    codes, scales, w, w_scale = make(m, n, k, seed=pad)
    wide_codes = torch.full((m, k + 32), -128, device="cuda", dtype=torch.int8)
    wide_codes[:, 16 : 16 + k] = codes
    buffer = torch.full((m + 2, n + pad), 7.0, device="cuda", dtype=torch.bfloat16)
    out = buffer[1 : m + 1, :n]
    got = kernels.w8a8_gemm(wide_codes[:, 16 : 16 + k], scales, w, w_scale, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_product(got, codes, scales, w, w_scale)
    assert (buffer[0] == 7).all() and (buffer[m + 1] == 7).all() and (buffer[:, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 70])
def test_longest_sum_of_the_largest_codes(m):
    k, n = 131056, 32
    codes = torch.full((m, k), -128, device="cuda", dtype=torch.int8)
    w = torch.full((n, k), -128, device="cuda", dtype=torch.int8)
    w[1] = 127
    ones = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    check_product(kernels.w8a8_gemm(codes, ones[0], w, ones[1]), codes, ones[0], w, ones[1])


@pytest.mark.gpu
def test_a_row_has_the_same_bits_in_every_batch():
    codes, scales, w, w_scale = make(2500, 4096, 1040)
    want = kernels.w8a8_gemm(codes, scales, w, w_scale)
    for m in (1, 16, 40, 64, 65, 300, 1000):
        assert torch.equal(kernels.w8a8_gemm(codes[:m], scales[:m], w, w_scale), want[:m])
    part = kernels.w8a8_gemm(codes[:300], scales[:300], w[:100], w_scale[:100])
    assert torch.equal(part, want[:300, :100])


@pytest.mark.gpu
def test_rows_and_outputs_past_32_bit_offsets():
    """2.3 10^9 codes and 4.5 10^9 outputs: the last rows have the bits that they have by themselves."""
    g = torch.Generator(device="cuda").manual_seed(3)
    m, k, n = 1_100_003, 2048, 4096
    x = torch.randn(40, k, device="cuda", generator=g).bfloat16()
    rows = x.repeat(m // 40 + 1, 1)[:m]
    codes, scales = kernels.quantize_rows(rows)
    del rows
    few = kernels.quantize_rows(x)
    order = torch.arange(m - 300, m, device="cuda") % 40
    assert torch.equal(codes[-300:], few[0][order]) and torch.equal(scales[-300:], few[1][order])
    w = torch.randint(-127, 128, (n, k), device="cuda", dtype=torch.int8, generator=g)
    ws = torch.rand(n, device="cuda", generator=g) * 0.01
    y = kernels.w8a8_gemm(codes, scales, w, ws)
    want = kernels.w8a8_gemm(*few, w, ws)
    for at in (0, (1 << 31) // n - 20, (1 << 32) // n - 20, m - 40):
        assert torch.equal(y[at : at + 40], want[torch.arange(at, at + 40, device="cuda") % 40])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 70, 700])
def test_weights_past_32_bit_offsets(m):
    g = torch.Generator(device="cuda").manual_seed(m)
    n, k = 33_000, 131_056
    w = torch.randint(-3, 4, (500, k), device="cuda", dtype=torch.int8, generator=g).repeat(n // 500, 1)
    ws = torch.rand(500, device="cuda", generator=g).repeat(n // 500) * 0.01
    codes = torch.randint(-127, 128, (m, k), device="cuda", dtype=torch.int8, generator=g)
    scales = torch.rand(m, device="cuda", generator=g)
    y = kernels.w8a8_gemm(codes, scales, w, ws).view(m, n // 500, 500)
    assert torch.equal(y, y[:, :1].expand_as(y))
    check_product(y[:, -1].contiguous(), codes, scales, w[:500], ws[:500])


def qkv_case(m, hq, hkv, k, cache, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, slots, spots = (hq + 2 * hkv) * 128, m + 9, 50
    codes, scales, w, w_scale = make(m, n, k, seed=seed)
    one = lambda: torch.randn(128, device="cuda", generator=g).bfloat16()
    i32 = lambda t: t.to(torch.int32)
    positions = i32(torch.randint(-2, spots + 3, (m,), device="cuda", generator=g))  # (clamped to the table)
    where = i32(torch.randperm(slots, device="cuda", generator=g)[:m])
    rope = (torch.rand(spots, 2, 64, device="cuda", generator=g) * 2 - 1).bfloat16()
    dtype, scale_dtype = cache
    def pool():
        caches = [torch.full((slots, hkv, 128), 7, device="cuda", dtype=dtype) for _ in range(2)]
        return caches + [torch.full((slots, hkv), 7, device="cuda", dtype=scale_dtype) if scale_dtype else None for _ in range(2)]
    return (codes, scales, w, w_scale), (one(), one(), 1e-6, positions, rope, where), pool


CACHES = [(torch.bfloat16, None), (torch.int8, torch.bfloat16), (torch.int8, torch.float16)]


@pytest.mark.gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("m,hq,hkv,k", [(1, 1, 1, 16), (5, 2, 1, 128), (130, 4, 2, 272), (300, 16, 8, 1024), (1000, 3, 1, 144),
                                        (4100, 16, 8, 128), (4001, 16, 8, 208), (22017, 3, 1, 128), (22017, 2, 2, 640)])
def test_qkv_product_is_the_two_calls_bits(m, hq, hkv, k, cache):
    """Queries, cache and its scales of the product fused with norm, rotation and write, against the
    product and the row kernel; slots that no row names stay as they were."""
    product_args, (q_norm, k_norm, eps, positions, rope, where), pool = qkv_case(m, hq, hkv, k, cache, seed=m + k)
    kc, vc, ks, vs = pool()
    want = kernels.qk_norm_rope_kv_write(kernels.w8a8_gemm(*product_args), hq, hkv, q_norm, k_norm, eps, positions, rope, where,
                                         kc, vc, ks, vs)
    got_pool = pool()
    q = torch.empty(m, hq, 128, device="cuda", dtype=torch.bfloat16)
    got = kernels.w8a8_qkv_norm_rope_kv(*product_args, hq, hkv, q_norm, k_norm, eps, positions, rope, where, *got_pool, q)
    assert got is q and torch.equal(q, want)
    for a, b in zip(got_pool, (kc, vc, ks, vs)):
        assert a is b is None or torch.equal(a, b)
    unnamed = torch.ones(m + 9, dtype=torch.bool, device="cuda")
    unnamed[where.long()] = False
    assert (got_pool[0][unnamed] == 7).all() and (got_pool[1][unnamed] == 7).all()


@pytest.mark.gpu
def test_qkv_product_of_strided_codes_replayed_on_another_stream():
    (codes, scales, w, w_scale), rest, pool = qkv_case(700, 4, 2, 256, CACHES[1])
    q_norm, k_norm, eps, positions, rope, where = rest
    wide = torch.zeros(700, 256 + 64, device="cuda", dtype=torch.int8)
    caches = pool()
    q = torch.empty(700, 4, 128, device="cuda", dtype=torch.bfloat16)
    call = lambda out, to: kernels.w8a8_qkv_norm_rope_kv(wide[:, :256], scales, w, w_scale, 4, 2, q_norm, k_norm, eps, positions,
                                                         rope, where, *to, out)
    call(q, caches)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q, caches)
    stream = torch.cuda.Stream()
    for step in range(3):
        wide[:, :256] = codes.roll(step, 0)
        positions.copy_(positions.roll(3))
        graph.replay()
        torch.cuda.synchronize()
        others, out = pool(), torch.empty_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            call(out, others)
        torch.cuda.synchronize()
        assert torch.equal(q, out) and all(torch.equal(a, b) for a, b in zip(caches, others))


@pytest.mark.gpu
def test_qkv_product_refuses_what_it_does_not_take():
    (codes, scales, w, w_scale), (q_norm, k_norm, eps, positions, rope, where), pool = qkv_case(6, 2, 1, 64, CACHES[1])
    kc, vc, ks, vs = pool()
    q = torch.empty(6, 2, 128, device="cuda", dtype=torch.bfloat16)
    good = dict(codes=codes, scales=scales, w_int8=w, w_scale=w_scale, num_q_heads=2, num_kv_heads=1, q_norm_weight=q_norm,
                k_norm_weight=k_norm, eps=eps, positions=positions, rope_cos_sin=rope, slot_mapping=where, k_cache=kc, v_cache=vc,
                k_scale=ks, v_scale=vs, q_out=q)
    for bad in (dict(codes=codes[:, :48]), dict(scales=scales[:5]), dict(w_int8=w[:128]), dict(num_q_heads=3),
                dict(q_norm_weight=q_norm.float()), dict(positions=positions.long()), dict(positions=positions[:5]),
                dict(slot_mapping=where[:5]), dict(rope_cos_sin=rope.float()), dict(q_out=q[:5]), dict(k_scale=None),
                dict(k_scale=ks[:3]), dict(v_cache=vc.bfloat16()), dict(v_scale=vs.half()), dict(w_scale=w_scale[:3])):
        with pytest.raises((ValueError, TypeError)):
            kernels.w8a8_qkv_norm_rope_kv(**{**good, **bad})
    with pytest.raises(_native.NativeError):
        kernels.w8a8_qkv_norm_rope_kv(**{**good, "k_scale": ks.float(), "v_scale": vs.float()})
    with pytest.raises(RuntimeError):
        kernels.w8a8_qkv_norm_rope_kv(**{**good, "positions": positions.cpu()})
    empty = {**good, "codes": codes[:0], "scales": scales[:0], "positions": positions[:0], "slot_mapping": where[:0], "q_out": q[:0]}
    assert kernels.w8a8_qkv_norm_rope_kv(**empty).shape == (0, 2, 128)


@pytest.mark.gpu
def test_no_rows():
    codes, scales, w, w_scale = make(4, 64, 64)
    assert kernels.w8a8_gemm(codes[:0], scales[:0], w, w_scale).shape == (0, 64)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    assert kernels.quantize_rows(x)[0].shape == (0, 64)
    assert kernels.rmsnorm_quantize(x, torch.ones(64, device="cuda", dtype=torch.bfloat16), 1e-6)[1].shape == (0,)


@pytest.mark.gpu
def test_captured_chain_follows_its_inputs_on_another_stream():
    """Norm, rows and product captured once and replayed on new rows, eager work in between."""
    m, n, k = 130, 768, 512
    _, _, w, w_scale = make(m, n, k)
    weight = torch.rand(k, device="cuda").bfloat16()
    x = torch.randn(m, k, device="cuda").bfloat16()
    codes, scales = torch.empty(m, k, device="cuda", dtype=torch.int8), torch.empty(m, device="cuda")
    out = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)

    def chain():
        kernels.rmsnorm_quantize(x, weight, 1e-6, codes=codes, scales=scales)
        kernels.w8a8_gemm(codes, scales, w, w_scale, out=out)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for seed in range(4):
        x.copy_(torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            chain()
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)
        check_product(out, codes, scales, w, w_scale)


@pytest.mark.gpu
def test_wrappers_refuse_what_the_kernels_do_not_take():
    codes, scales, w, w_scale = make(4, 64, 64)
    bf = dict(device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        kernels.w8a8_gemm(codes[:, :48], scales, w, w_scale)
    with pytest.raises(ValueError):
        kernels.w8a8_gemm(codes, scales[:3], w, w_scale)
    with pytest.raises(ValueError):
        kernels.w8a8_gemm(codes, scales.double(), w, w_scale)
    with pytest.raises(ValueError):
        kernels.w8a8_gemm(codes, scales, w, w_scale[:10])
    with pytest.raises(ValueError):
        kernels.w8a8_gemm(codes, scales, w, w_scale, out=torch.empty(4, 63, **bf))
    with pytest.raises(RuntimeError):
        kernels.w8a8_gemm(codes.cpu(), scales, w, w_scale)
    with pytest.raises(_native.NativeError):  # k off 16
        kernels.w8a8_gemm(codes[:, :40].contiguous(), scales, w[:, :40].contiguous(), w_scale)
    with pytest.raises(_native.NativeError):  # codes off 16 bytes
        kernels.w8a8_gemm(codes[:, 8:56], scales, w[:, :48].contiguous(), w_scale)
    with pytest.raises(_native.NativeError):
        kernels.w8a8_gemm(codes, scales, w[:48].contiguous(), w_scale[:48], epilogue=EPILOGUE_SWIGLU)
    with pytest.raises(ValueError):
        kernels.quantize_rows(torch.ones(4, 64, device="cuda"))
    with pytest.raises(_native.NativeError):
        kernels.quantize_rows(torch.ones(4, 60, **bf))
    with pytest.raises(_native.NativeError):
        kernels.quantize_rows(torch.ones(4, 72, **bf)[:, 4:68])
    with pytest.raises(ValueError):
        kernels.quantize_rows(torch.ones(4, 64, **bf), codes=torch.empty(4, 64, device="cuda"))
    with pytest.raises(ValueError):
        kernels.rmsnorm_quantize(torch.ones(4, 64, **bf), torch.ones(32, **bf), 1e-6)
    with pytest.raises(_native.NativeError):
        kernels.rmsnorm_quantize(torch.ones(4, 4104, **bf), torch.ones(4104, **bf), 1e-6)


def test_entry_points_refuse_bad_arguments_without_launching():
    if not _native.library_path().exists():
        pytest.skip("libnanoengine_hip.so is not built")
    lib = _native.load()
    p, odd, null = ctypes.c_void_p(256), ctypes.c_void_p(264), ctypes.c_void_p(0)

    def gemm(x=p, ldx=64, xs=p, w=p, ws=p, dt=0, m=4, n=64, k=64, y=p, ldy=64, epilogue=0):
        return lib.ne_w8a8_gemm(x, ldx, xs, w, ws, dt, m, n, k, y, ldy, epilogue, null)

    assert gemm(m=0, x=null) == 0
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(epilogue=7), dict(dt=3), dict(x=null), dict(xs=null), dict(ws=null),
                dict(y=null), dict(x=odd), dict(w=odd), dict(ldx=48), dict(ldx=72), dict(ldx=1 << 23), dict(ldy=63),
                dict(xs=ctypes.c_void_p(258)), dict(ws=ctypes.c_void_p(257)), dict(ws=ctypes.c_void_p(258), dt=2),
                dict(y=ctypes.c_void_p(257))):
        assert gemm(**bad) == -1, bad
    for bad in (dict(k=72, ldx=80), dict(k=131072, ldx=131072), dict(epilogue=1, n=48), dict(m=(1 << 30) + 1),
                dict(n=(1 << 30) + 1, ldy=1 << 31)):
        assert gemm(**bad) == -2, bad

    def qkv(x=p, ldx=64, xs=p, w=p, ws=p, dt=0, m=4, hq=2, hkv=1, k=64, qn=p, kn=p, pos=p, rope=p, spots=8, slots=p, kv=3, kc=p, vc=p,
            ks=p, vs=p, sdt=0, q=p):
        return lib.ne_w8a8_qkv_norm_rope_kv(x, ldx, xs, w, ws, dt, m, hq, hkv, k, qn, kn, 1e-6, pos, rope, spots, slots, kv, kc, vc, ks,
                                            vs, sdt, q, null)

    assert qkv(m=0, x=null) == 0
    byte8, byte2 = ctypes.c_void_p(264), ctypes.c_void_p(258)
    for bad in (dict(m=-1), dict(hq=0), dict(hkv=-1), dict(hq=1 << 21), dict(k=0), dict(dt=3), dict(x=null), dict(xs=null),
                dict(ws=null), dict(x=odd), dict(w=odd), dict(ldx=72), dict(qn=null), dict(kn=byte2), dict(pos=null), dict(rope=null),
                dict(rope=ctypes.c_void_p(260)), dict(spots=0), dict(slots=null), dict(kv=2), dict(kc=null), dict(vc=byte8),
                dict(ks=null), dict(q=null), dict(q=byte8)):
        assert qkv(**bad) == -1, bad
    for bad in (dict(k=72, ldx=80), dict(sdt=2), dict(m=(1 << 30) + 1)):
        assert qkv(**bad) == -2, bad
    assert lib.ne_quantize_rows(p, 0, 64, 0, 64, null, null, null) == 0
    assert lib.ne_quantize_rows(p, 2, 64, 4, 64, p, p, null) == -1
    assert lib.ne_quantize_rows(p, 0, 60, 4, 64, p, p, null) == -1
    assert lib.ne_quantize_rows(odd, 0, 64, 4, 64, p, p, null) == -1
    assert lib.ne_quantize_rows(p, 0, 64, 4, 60, p, p, null) == -2
    assert lib.ne_quantize_rows(null, 0, 64, 4, 64, p, p, null) == -1
    for rows, k in ((1 << 26, 8), (1 << 26, 2048), (1 << 24, 4096), (1 << 24, 4104), (1 << 22, 16392)):  # 2^32 threads
        assert lib.ne_quantize_rows(p, 0, k, rows, k, p, p, null) == -2
    assert lib.ne_rmsnorm_quantize(p, p, p, p, 1 << 26, 64, 1e-6, null) == -2
    assert lib.ne_rmsnorm_quantize(p, null, p, p, 4, 64, 1e-6, null) == -1
    assert lib.ne_rmsnorm_quantize(p, p, p, p, 4, 4104, 1e-6, null) == -2
    assert lib.ne_add_rmsnorm_quantize(p, odd, p, p, p, 4, 64, 1e-6, null) == -1
