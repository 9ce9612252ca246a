// W8A8 products for gfx950: y[m, n] = bf16((sum_k q[m, k] w[n, k]) s[m] t[n]) for rows of 8-bit
// activations q with one scale each (quantize_rows.hip) and the int8 weights and row scales
// that the W8A16 products read.  The sum is exact in int32 (k <= 131,056 holds any codes), so
// no result depends on how k is split or ordered: every kernel here gives the same bits.
//
// As in gemm.hip an MFMA computes D = W . X^T (v_mfma_i32_16x16x64_i8), so that a lane holds
// four consecutive output columns of one token row.
#include "ne_common.hpp"
#include "qk_rope_kv.hpp"

namespace ne {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));

struct W8a8Params {
  const int8_t* x;  // codes [m][ldx]
  int64_t ldx;
  const float* xs;  // [m]
  const int8_t* w;  // [n][k]
  const void* ws;   // [n]
  int ws_dtype;
  int m, n, k;
  uint16_t* y;
  int64_t ldy;
  int tiles_m, tiles_n;
};

// the product's rows as head vectors, through QK-norm and RoPE into q_out and the KV cache
constexpr int kEpilogueQkvBf16 = 2, kEpilogueQkvInt8 = 3;  // (by the cache's type)
struct W8a8QkvParams : W8a8Params {
  QkvRopeArgs qkv;
  int kv_scale_dtype;
};
template <bool QKV>
struct ParamsFor {
  using type = W8a8Params;
};
template <>
struct ParamsFor<true> {
  using type = W8a8QkvParams;
};
template <int EPI>
using ParamsOf = typename ParamsFor<(EPI >= 2)>::type;  // (a kernel's name spells this out: literals only)

__device__ __forceinline__ void lds_dma16(const void* src, void* lds_wave_base) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

__device__ __forceinline__ void lds_dma4(const void* src, void* lds_wave_base) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds_wave_base, 4, 0, 0);
}

// s_waitcnt vmcnt(n) leaving lgkmcnt/expcnt unconstrained (gfx9 encoding)
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }

// s_waitcnt vmcnt(D * pend) for a run-time pend in [0, P]
template <int D, int P>
__device__ __forceinline__ void wait_pending(int pend) {
  if constexpr (P <= 0) {
    wait_vmcnt<0>();
  } else {
    if (pend >= P) {
      wait_vmcnt<D * P>();
    } else {
      wait_pending<D, P - 1>(pend);
    }
  }
}

// the same with S younger stores in flight
template <int D, int P, int S>
__device__ __forceinline__ void wait_pending_after(int pend) {
  if constexpr (P <= 0) {
    wait_vmcnt<S>();
  } else {
    if (pend >= P) {
      wait_vmcnt<D * P + S>();
    } else {
      wait_pending_after<D, P - 1, S>(pend);
    }
  }
}

__device__ __forceinline__ const char* uniform_ptr(const char* ptr) {
  const uint64_t v = (uint64_t)ptr;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)(((uint64_t)hi << 32) | lo);
}

// scale of weight row i in the caller's dtype (a uniform branch)
__device__ __forceinline__ float weight_scale(const W8a8Params& p, int i) {
  if (p.ws_dtype == NE_DTYPE_BF16) return load_scale<NE_DTYPE_BF16>(p.ws, i);
  if (p.ws_dtype == NE_DTYPE_FP16) return load_scale<NE_DTYPE_FP16>(p.ws, i);
  return load_scale<NE_DTYPE_FP32>(p.ws, i);
}

__device__ __forceinline__ u32x2 store4(const intx4& v, float s, const float (&t)[4]) {
  return u32x2{pack_bf16x2((float)v[0] * s * t[0], (float)v[1] * s * t[1]),
               pack_bf16x2((float)v[2] * s * t[2], (float)v[3] * s * t[3])};
}

// silu(gate) * up in fp32, rounded once
__device__ __forceinline__ u32x2 swiglu4(const intx4& gate, const intx4& up, float s, const float (&gt)[4],
                                         const float (&ut)[4]) {
  float out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = (float)gate[i] * s * gt[i];
    out[i] = a / (1.f + __expf(-a)) * ((float)up[i] * s * ut[i]);
  }
  return u32x2{pack_bf16x2(out[0], out[1]), pack_bf16x2(out[2], out[3])};
}

// Two adjacent 16-column subtiles of a row, lane group g with columns 4 g .. + 4 of each:
// regrouped so that the lane holds 8 consecutive columns from pair_column(g) on.
__device__ __forceinline__ u32x4 pair_columns(const u32x2& a, const u32x2& b) {
  const auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{x[0], y[0], x[1], y[1]};
}
__device__ __forceinline__ int pair_column(int g) { return 16 * (g & 1) + 8 * (g >> 1); }

// ---- the QKV epilogue's arithmetic: what qk_norm_rope_kv_vectors does, bit for bit for finite rows ----
// A lane holds columns 16 ns + 4 g + i (ns < 8, i < 4) of a row's 128, its RoPE pairs 64 apart
// among them; a vector's sums are taken in the row kernel's order.
__device__ __forceinline__ float plain_add(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}
__device__ __forceinline__ float add_xor16(float v) {
  const auto o = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return plain_add(__uint_as_float(o[0]), __uint_as_float(o[1]));
}
__device__ __forceinline__ float add_xor32(float v) {
  const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return plain_add(__uint_as_float(o[0]), __uint_as_float(o[1]));
}
__device__ __forceinline__ uint32_t max_over_groups(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}
__device__ __forceinline__ float lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// 1 / rms of a row: the squares of each 16 columns and their partners, then the tree over 64 lanes
__device__ __forceinline__ float inverse_rms(const u32x2 (&v)[8], float eps) {
  float sums[4];
#pragma unroll
  for (int ns = 0; ns < 4; ++ns) {
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = i % 2 ? hi_f32(v[ns][i / 2]) : lo_f32(v[ns][i / 2]);
      const float b = i % 2 ? hi_f32(v[ns + 4][i / 2]) : lo_f32(v[ns + 4][i / 2]);
      t[i] = a * a + b * b;
    }
    sums[ns] = add_xor32(add_xor16(plain_add(plain_add(t[0], t[1]), plain_add(t[2], t[3]))));
  }
  return rsqrtf(plain_add(plain_add(sums[0], sums[1]), plain_add(sums[2], sums[3])) / 128.f + eps);
}

// two neighbouring columns of each half: norm, then rotation, in place
__device__ __forceinline__ void norm_rope2(uint32_t& a, uint32_t& b, float inv, uint32_t wa, uint32_t wb, uint32_t c, uint32_t s) {
  uint32_t x = pack_bf16x2(lo_f32(a) * inv, hi_f32(a) * inv), y = pack_bf16x2(lo_f32(b) * inv, hi_f32(b) * inv);
  x = pack_bf16x2(lo_f32(x) * lo_f32(wa), hi_f32(x) * hi_f32(wa));
  y = pack_bf16x2(lo_f32(y) * lo_f32(wb), hi_f32(y) * hi_f32(wb));
  const uint32_t xc = pack_bf16x2(lo_f32(x) * lo_f32(c), hi_f32(x) * hi_f32(c));
  const uint32_t ys = pack_bf16x2(-lo_f32(y) * lo_f32(s), -hi_f32(y) * hi_f32(s));
  const uint32_t yc = pack_bf16x2(lo_f32(y) * lo_f32(c), hi_f32(y) * hi_f32(c));
  const uint32_t xs = pack_bf16x2(lo_f32(x) * lo_f32(s), hi_f32(x) * hi_f32(s));
  a = pack_bf16x2(lo_f32(xc) + lo_f32(ys), hi_f32(xc) + hi_f32(ys));
  b = pack_bf16x2(lo_f32(yc) + lo_f32(xs), hi_f32(yc) + hi_f32(xs));
}

// a row's scale and the codes of this lane's columns, four in a word (as quantize_rows.hip's: the
// quotients' own, by division only in waves with one next to a half)
__device__ __forceinline__ float quantize_vector(const u32x2 (&v)[8], uint32_t (&codes)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int ns = 0; ns < 8; ++ns)
#pragma unroll
    for (int i = 0; i < 2; ++i) top = max(top, max(v[ns][i] << 16 & 0x7FFF0000u, v[ns][i] & 0x7FFF0000u));
  const float s = fmaxf(__uint_as_float(max_over_groups(top)), 1e-8f) / 127.f;
  const float rcp = __builtin_amdgcn_rcpf(s);
  constexpr float kWhole = 12582912.f;  // 1.5 2^23
#pragma unroll
  for (int ns = 0; ns < 8; ++ns) {
    const float f[4] = {lo_f32(v[ns][0]), hi_f32(v[ns][0]), lo_f32(v[ns][1]), hi_f32(v[ns][1])};
    float t[4], far = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = __builtin_fmaf(f[e], rcp, kWhole);
      far = fmaxf(far, fabsf(__builtin_fmaf(f[e], rcp, -(t[e] - kWhole))));
    }
    if (__builtin_amdgcn_ballot_w64(far > 0.49996f) != 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = f[e] / s + kWhole;
    }
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[1]), __float_as_uint(t[0]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[3]), __float_as_uint(t[2]), 0x0c0c0400u);
    codes[ns] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return s;
}

// words j of lane group g to word g of lane group j: lane group g then holds subtile g's 16 columns
__device__ __forceinline__ u32x4 transpose_groups(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const auto ab = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  const auto cd = __builtin_amdgcn_permlane16_swap(c, d, false, false);
  const auto even = __builtin_amdgcn_permlane32_swap(ab[0], cd[0], false, false);
  const auto odd = __builtin_amdgcn_permlane32_swap(ab[1], cd[1], false, false);
  return u32x4{even[0], odd[0], even[1], odd[1]};
}

// columns col .. + 2 N of a row of n_out, element by element where the row's end or the
// alignment does not take a wide store
template <int N, typename V>
__device__ __forceinline__ void store_columns(uint16_t* row, int col, int n_out, bool wide, const V& v) {
  if (wide && col + 2 * N <= n_out) {
    *(V*)(row + col) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (col + 2 * i < n_out) row[col + 2 * i] = (uint16_t)(v[i] & 0xFFFFu);
    if (col + 2 * i + 1 < n_out) row[col + 2 * i + 1] = (uint16_t)(v[i] >> 16);
  }
}

// ---- many rows: tiles through LDS --------------------------------------------------
//   stage = 128 k of BM rows and BN weight rows (whole 128-byte lines), copied by DMA
//           (global_load_lds_dwordx4), the 16-byte chunks of a row swizzled so that the fragment
//           reads are free of bank conflicts
//   ring  = RING stages; a wave holds the next k-step's fragments while the MFMAs of the current
//           one run, and the barrier that admits a stage sits between two batches of MFMAs
//   tiles = a work-group walks several, its stages run on across them: the next tile's first
//           stages are on their way while a tile is scaled, rounded and stored
// 256 x 256 tiles, 8,192 cubed: 420-458 us, 2.4-2.6 POP/s (the library's int8 product, without
// scales and into int32, 514): MFMA busy 61 % at a clock that the power limit holds near 1.7 GHz, no
// LDS bank conflicts.  64-byte lines instead of 128 took 836 us, one wave per SIMD (128 x 128 a wave)
// 705.  8,192 x 4,096 x 1,024: 40 us, of which 13 store y; without the walk over tiles 43.
// 128 x 128 tiles, one per CU (4,001 x 1,024 x 2,048): 17.8 us, 5.7 fixed and 0.75 a stage: MFMAs and
// barriers 0.35, fragment reads 0.13 (64 KB a stage, as long as the MFMAs), copies 0.27 more.  Rings of
// three and four stages, eight waves, a second set of waves on the other half of every stage's k
// and copies spread over both halves of a stage were within 5 % of it or slower.
template <int BM_, int BN_, int MW_, int NW_, int RING_>
struct TileLayout {
  static constexpr int BM = BM_, BN = BN_, MW = MW_, NW = NW_, RING = RING_;
  static constexpr int kWaves = MW * NW;
  static constexpr int PM = BM / MW / 16;   // token subtiles per wave
  static constexpr int NPW = BN / NW / 16;  // weight subtiles per wave
  static constexpr int kStage = (BM + BN) * 128;
  static constexpr int kCopies = kStage / 1024 / kWaves;  // per wave and stage
  static constexpr int kXCopies = BM / 8 / kWaves;
  static constexpr int kScales = RING * kStage;  // LDS: the ring, then BM + BN scales
  static constexpr int kEdge = kScales + (BM + BN) * 4;  // then 1 KiB per wave for tiles at an edge
  static constexpr int kLds = kEdge + kWaves * 1024;
  static constexpr int kPerCu = 160 * 1024 / kLds;  // work-groups
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "copies split evenly over the waves");
  static_assert(BM + BN <= kWaves * kWave, "a scale per thread");
  static_assert(RING >= 2 && kPerCu >= 1, "ring");
};

template <typename L, int EPI>
__global__ __launch_bounds__(L::kWaves* kWave) void w8a8_tile_kernel(ParamsOf<EPI> p) {
  constexpr int PM = L::PM, NPW = L::NPW, RING = L::RING, D = L::kCopies;
  constexpr int kOut = EPI == NE_EPILOGUE_SWIGLU ? NPW / 2 : NPW;
  constexpr bool kQkv = EPI >= kEpilogueQkvBf16;
  constexpr int kStores = EPI == kEpilogueQkvInt8 ? PM * 2 : PM * kOut / 2;  // of a wave's whole tile, at least
  static_assert(!kQkv || L::BN == 128 * L::NW, "a wave's columns are a head");
  static_assert(D * (RING - 1) + kStores < 64, "vmcnt range");
  __shared__ __attribute__((aligned(16))) char smem[L::kLds + (kQkv ? L::BM * 16 : 0)];
  float* const scales = (float*)(smem + L::kScales);
  // Each XCD takes a contiguous eighth of the tiles, in an order that walks all weight tiles
  // against groups of four row tiles: the group's rows stay in that XCD's L2.  Its work-groups
  // take them in turn.
  const int total = p.tiles_m * p.tiles_n;
  const int per = (total + kNumXcd - 1) / kNumXcd;
  const int base = (int)(blockIdx.x % kNumXcd) * per;
  const int here = max(min(per, total - base), 0);  // tiles of this XCD
  const int first = blockIdx.x / kNumXcd, step = gridDim.x / kNumXcd;
  if (first >= here) return;
  const int my_tiles = (here - 1 - first) / step + 1;
  auto place = [&](int i, int& m0, int& n0) {
    const int idx = base + first + i * step;
    constexpr int kGroup = 4;
    const int grp = idx / (kGroup * p.tiles_n);
    const int in_grp = idx - grp * kGroup * p.tiles_n;
    const int rows_in = min(kGroup, p.tiles_m - grp * kGroup);
    const int tn = in_grp / rows_in;
    m0 = (grp * kGroup + in_grp - tn * rows_in) * L::BM;
    n0 = tn * L::BN;
  };
  const int lane = threadIdx.x % kWave;
  const int r = lane & 15;
  const int g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int mw = wave / L::NW, nw = wave % L::NW;
  const int n_stages = (p.k + 127) / 128;  // per tile
  const int all = my_tiles * n_stages;

  // Copy j of this wave is KiB j kWaves + wave of the stage, eight rows: token rows, then weight
  // rows.  LDS row `row` holds chunk c at position c ^ (row % 8), and row % 8 is lane / 8 in every
  // copy.  Rows past m and n re-read the last one and are never stored; chunks past k re-read the
  // last one, and the token rows' are then zeroed in LDS.
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;  // bytes
  const uint32_t xrow = (uint32_t)(wave * 8 + (lane >> 3)) * (uint32_t)p.ldx;
  const uint32_t wrow = (uint32_t)(wave * 8 + (lane >> 3)) * (uint32_t)p.k;
  uint32_t xlast = 0, wlast = 0;  // of the last rows
  const char *xbase = nullptr, *wbase = nullptr;
  int next_tile = 0, next_stage = 0;  // of the copies
  char* next_slot = smem;
  int column = 0;
  auto begin_copies = [&]() {
    if (next_stage == 0) {
      int m0, n0;
      place(next_tile, m0, n0);
      xbase = uniform_ptr((const char*)p.x + (int64_t)m0 * p.ldx);
      wbase = uniform_ptr((const char*)p.w + (int64_t)n0 * p.k);
      xlast = (uint32_t)(min(p.m - m0, L::BM) - 1) * (uint32_t)p.ldx;
      wlast = (uint32_t)(min(p.n - n0, L::BN) - 1) * (uint32_t)p.k;
    }
    column = chunk - max(next_stage * 128 + chunk - (p.k - 16), 0);
  };
  auto copies = [&](int from, int to) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      if (j < from || j >= to) continue;
      const uint32_t rows = (uint32_t)((j < L::kXCopies ? j : j - L::kXCopies) * L::kWaves * 8);
      uint32_t o = (j < L::kXCopies ? min(xrow + rows * (uint32_t)p.ldx, xlast) : min(wrow + rows * (uint32_t)p.k, wlast)) + column;
      __asm__("" : "+v"(o));  // keep the lane offset 32-bit: scalar base + offset addressing
      lds_dma16((j < L::kXCopies ? xbase : wbase) + o, next_slot + (j * L::kWaves + wave) * 1024);
    }
  };
  auto end_copies = [&]() {
    xbase += 128;
    wbase += 128;
    next_slot = next_slot == smem + (RING - 1) * L::kStage ? smem : next_slot + L::kStage;
    if (++next_stage == n_stages) {
      next_stage = 0;
      ++next_tile;
    }
  };

  auto issue = [&]() {
    begin_copies();
    copies(0, D);
    end_copies();
  };

  struct Frags {
    intx4 x[PM], w[NPW];
  };
  // chunk 4 q + g of a row sits at position chunk ^ (row % 8); rows 16 apart swizzle alike
  auto read = [&](const char* slot, int q, Frags& f) {
    const char* at = slot + (((4 * q + g) ^ (r & 7)) * 16 + r * 128);
#pragma unroll
    for (int ns = 0; ns < NPW; ++ns) f.w[ns] = *(const intx4*)(at + (L::BM + (nw * NPW + ns) * 16) * 128);
#pragma unroll
    for (int mi = 0; mi < PM; ++mi) f.x[mi] = *(const intx4*)(at + (mw * PM + mi) * 16 * 128);
  };
  // zeroes this wave's own copies of token chunks past k in a landed stage
  auto clear_tail = [&](char* slot, int stage) {
    if (stage * 128 + 128 > p.k && stage * 128 + chunk >= p.k) {
#pragma unroll
      for (int j = 0; j < L::kXCopies; ++j) *(intx4*)(slot + (j * L::kWaves + wave) * 1024 + lane * 16) = intx4{0, 0, 0, 0};
    }
  };
  intx4 acc[PM][NPW];
  auto mma_row = [&](const Frags& f, int mi) {
#pragma unroll
    for (int ns = 0; ns < NPW; ++ns)
      acc[mi][ns] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[ns], f.x[mi], acc[mi][ns], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto mma = [&](const Frags& f) {
    __builtin_amdgcn_sched_barrier(0);  // the reads before it go out first
#pragma unroll
    for (int mi = 0; mi < PM; ++mi) mma_row(f, mi);
  };

#pragma unroll 1
  for (int s = 0; s < min(RING, all); ++s) issue();
  wait_pending<D, RING - 1>(min(all, RING) - 1);  // stage 0 has landed
  clear_tail(smem, 0);
  wait_lgkmcnt0();
  asm volatile("s_barrier" ::: "memory");

  Frags a, b;
  char* slot = smem;
  int s = 0;             // stage over all tiles
  bool storing = false;  // the previous tile's kStores stores are younger than the copies up to stage s + RING - 1
  const bool wide = (uintptr_t)p.y % 16 == 0 && p.ldy % 8 == 0;
  const int n_out = EPI == NE_EPILOGUE_SWIGLU ? p.n / 2 : p.n;
#pragma unroll 1
  for (int i = 0; i < my_tiles; ++i) {
    int m0, n0;
    place(i, m0, n0);
    // the bits of this thread's scale, one of BM + BN, so that nothing waits for them where they are loaded
    auto my_scale = [&]() -> uint32_t {
      int t = threadIdx.x;
      if constexpr (kQkv) __asm__ volatile("" : "+v"(t));  // its registers are for the QKV epilogue
      if (t < L::BM) return ((const uint32_t*)p.xs)[min(m0 + t, p.m - 1)];
      const int n = min(n0 + min(t - L::BM, L::BN - 1), p.n - 1);
      return p.ws_dtype == NE_DTYPE_FP32 ? ((const uint32_t*)p.ws)[n] : ((const uint16_t*)p.ws)[n];
    };
    auto put_scale = [&](uint32_t bits) {
      int t = threadIdx.x;
      if constexpr (kQkv) __asm__ volatile("" : "+v"(t));
      const bool fp32 = t < L::BM || p.ws_dtype == NE_DTYPE_FP32;
      const float half = p.ws_dtype == NE_DTYPE_BF16 ? bf16_to_f32((uint16_t)bits) : f16_to_f32((uint16_t)bits);
      const float v = fp32 ? __uint_as_float(bits) : half;
      if (L::BM + L::BN == L::kWaves * kWave || t < L::BM + L::BN) scales[t] = v;
    };
    uint32_t scale = 0;
    const int head = n0 / 128 + nw;  // QKV
    int* const places = (int*)(smem + L::kLds) + (i & 1) * 2 * L::BM;  // QKV: the rows' positions, then their slots
#pragma unroll
    for (int mi = 0; mi < PM; ++mi)
#pragma unroll
      for (int ns = 0; ns < NPW; ++ns) acc[mi][ns] = intx4{0, 0, 0, 0};
    read(slot, 0, a);
#pragma unroll 1
    for (int t = 0; t < n_stages; ++t, ++s) {
      wait_lgkmcnt0();  // for a's reads, not for the next ones too
      read(slot, 1, b);
      if (t + 1 == n_stages) {
        if constexpr (kQkv) {
          // by DMA, as they are wanted next to no registers: a wave's 64 rows, and its head's norm weights
          static_assert(RING == 2 && L::BM % kWave == 0 && L::BM / kWave <= L::kWaves, "rows by waves");
          int l = lane;
          __asm__ volatile("" : "+v"(l));
          if (wave < L::BM / kWave) {
            const int m = min(m0 + wave * kWave + l, p.m - 1);
            lds_dma4(p.qkv.positions + m, places + wave * kWave);
            lds_dma4(p.qkv.slot_mapping + m, places + L::BM + wave * kWave);
          }
          lds_dma4((const uint32_t*)(head < p.qkv.hq ? p.qkv.q_norm_w : p.qkv.k_norm_w) + l, smem + L::kEdge + wave * 1024);
        }
        scale = my_scale();
      }
      mma(a);
      if (s + 1 < all) {
        // stage s + 1 has landed and every wave has read all of stage s: its slot takes stage s + RING
        const int pend = min(all - 1, s + RING - 1) - (s + 1);
        if (storing && t <= RING - 2) {
          wait_pending_after<D, RING - 2, kStores>(pend);
        } else {
          wait_pending<D, RING - 2>(pend);
        }
        slot = slot == smem + (RING - 1) * L::kStage ? smem : slot + L::kStage;
        clear_tail(slot, t + 1 == n_stages ? 0 : t + 1);
        wait_lgkmcnt0();
        asm volatile("s_barrier" ::: "memory");
        if (t + 1 < n_stages) read(slot, 0, a);
      } else {
        wait_lgkmcnt0();
      }
      // the next copies go out between the MFMAs, which hide them
      const bool more = s + RING < all && t + 1 < n_stages;
      if (more) begin_copies();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int mi = 0; mi < PM; ++mi) {
        mma_row(b, mi);
        if (more) copies(D * mi / PM, D * (mi + 1) / PM);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (more) end_copies();
    }
    // The scales go through LDS.  Their load is waited for before the copies of the slot that the
    // tile's last stage left, not after them.
    if (n_stages == 1) lds_barrier();  // the previous tile's have been read
    put_scale(scale);
    if constexpr (kQkv) wait_vmcnt<0>();  // (no copies are in flight here)
    if (s - 1 + RING < all) issue();
    lds_barrier();

    // lane (r, g): rows 16 mi + r, columns 16 ns + 4 g + i
    int l = lane;
    __asm__ volatile("" : "+v"(l));  // addresses made here, not kept in registers through the k loop
    const int er = l & 15, eg = l >> 4;
    if constexpr (kQkv) {
      const QkvRopeArgs& qa = p.qkv;
      const bool is_q = head < qa.hq, is_v = head >= qa.hq + qa.hkv;
      const bool is_head = head < qa.hq + 2 * qa.hkv;  // (the last tile's other half may be none)
      const int kv_head = head - qa.hq - (is_v ? qa.hkv : 0);
      const char* const norm = smem + L::kEdge + wave * 1024;
      void* const cache = is_v ? qa.v_cache : qa.k_cache;
      u32x2 rope[8];  // cosines and sines of this lane's columns
      auto load_rope = [&](int mi) {
        const uint16_t* at = qa.rope + (int64_t)min(max(places[(mw * PM + mi) * 16 + er], 0), qa.rope_positions - 1) * 128 + 4 * eg;
#pragma unroll
        for (int ns = 0; ns < 4; ++ns) {
          rope[ns] = *(const u32x2*)(at + 16 * ns);
          rope[4 + ns] = *(const u32x2*)(at + 64 + 16 * ns);
        }
      };
      if (is_head) {
        load_rope(0);  // (also for v, which has no use for them: fewer registers than a choice)
#pragma unroll
        for (int mi = 0; mi < PM; ++mi) {
          const int lrow = (mw * PM + mi) * 16 + er;
          const float sx = scales[lrow];
          const bool real = m0 + lrow < p.m;
          u32x2 v[8];
#pragma unroll
          for (int ns = 0; ns < 8; ++ns) {
            const floatx4 sc = *(const floatx4*)(scales + L::BM + (nw * 8 + ns) * 16 + 4 * eg);
            v[ns] = store4(acc[mi][ns], sx, {sc[0], sc[1], sc[2], sc[3]});
          }
          if (!is_v) {
            const float inv = inverse_rms(v, qa.eps);
#pragma unroll
            for (int ns = 0; ns < 4; ++ns) {
              const u32x2 wa = *(const u32x2*)(norm + (16 * ns + 4 * eg) * 2), wb = *(const u32x2*)(norm + (64 + 16 * ns + 4 * eg) * 2);
              const u32x2 c = rope[ns], sn = rope[4 + ns];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t x = v[ns][i], y = v[ns + 4][i];
                norm_rope2(x, y, inv, wa[i], wb[i], c[i], sn[i]);
                v[ns][i] = x;
                v[ns + 4][i] = y;
              }
            }
          }
          if (mi + 1 < PM) load_rope(mi + 1);
          const int64_t vector = (int64_t)places[L::BM + lrow] * qa.hkv + kv_head;  // in the cache
          if (EPI == kEpilogueQkvBf16 || is_q) {
            uint16_t* to = is_q ? qa.q_out + ((int64_t)(m0 + lrow) * qa.hq + head) * 128 : (uint16_t*)cache + vector * 128;
#pragma unroll
            for (int o = 0; o < 8; o += 2) {
              const u32x4 both = pair_columns(v[o], v[o + 1]);
              if (real) *(u32x4*)(to + o * 16 + pair_column(eg)) = both;
            }
          } else {
            uint32_t codes[8];
            const float sv = quantize_vector(v, codes);
            const u32x4 low = transpose_groups(codes[0], codes[1], codes[2], codes[3]);
            const u32x4 high = transpose_groups(codes[4], codes[5], codes[6], codes[7]);
            int8_t* to = (int8_t*)cache + vector * 128 + 16 * eg;
            if (real) {
              *(u32x4*)to = low;
              *(u32x4*)(to + 64) = high;
              if (eg == 0) {
                void* const kv_scales = is_v ? qa.v_scale : qa.k_scale;
                if (p.kv_scale_dtype == NE_DTYPE_BF16) {
                  store_scale<NE_DTYPE_BF16>(kv_scales, vector, sv);
                } else {
                  store_scale<NE_DTYPE_FP16>(kv_scales, vector, sv);
                }
              }
            }
          }
        }
      }
      storing = is_head && m0 + L::BM <= p.m;
    } else {
      float sc[NPW][4];
#pragma unroll
      for (int ns = 0; ns < NPW; ++ns) {
        const floatx4 v = *(const floatx4*)(scales + L::BM + (nw * NPW + ns) * 16 + 4 * eg);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[ns][e] = v[e];
      }
      const int col0 = (EPI == NE_EPILOGUE_SWIGLU ? n0 / 2 : n0) + nw * kOut * 16;
      const bool inside = wide && n0 + L::BN <= p.n;  // all of the tile's columns, in wide stores
      auto out4 = [&](int mi, int o, float sx) {
        if constexpr (EPI == NE_EPILOGUE_SWIGLU)
          return swiglu4(acc[mi][2 * o], acc[mi][2 * o + 1], sx, sc[2 * o], sc[2 * o + 1]);
        else
          return store4(acc[mi][o], sx, sc[o]);
      };
      char* const edge = smem + L::kEdge + wave * 1024;
#pragma unroll
      for (int mi = 0; mi < PM; ++mi) {
        const int lrow = (mw * PM + mi) * 16 + er;
        const float sx = scales[lrow];
        uint16_t* row = p.y + (int64_t)(m0 + lrow) * p.ldy + col0;
        // a row's 16-column subtiles in pairs
        static_assert(kOut % 2 == 0, "output subtiles in pairs");
#pragma unroll
        for (int o = 0; o < kOut; o += 2) {
          const u32x4 both = pair_columns(out4(mi, o, sx), out4(mi, o + 1, sx));
          if (inside) {
            if (m0 + lrow < p.m) *(u32x4*)(row + o * 16 + pair_column(eg)) = both;
          } else {
            // 16 rows of 32 columns through LDS, then two rows at a time, element by element
            *(u32x4*)(edge + er * 64 + pair_column(eg) * 2) = both;
#pragma unroll 1
            for (int at = l; at < 16 * 32; at += kWave) {
              const int m = m0 + (mw * PM + mi) * 16 + at / 32, col = col0 + o * 16 + at % 32;
              if (m < p.m && col < n_out) p.y[(int64_t)m * p.ldy + col] = *(const uint16_t*)(edge + at * 2);
            }
          }
        }
      }
      storing = inside && m0 + L::BM <= p.m;  // (every one of the stores was made)
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);  // the stores stay before the next wait
  }
}

template <typename L, int EPI>
int launch_tile(ParamsOf<EPI> p, hipStream_t stream) {
  p.tiles_m = ceil_div(p.m, L::BM);
  p.tiles_n = ceil_div(p.n, L::BN);
  const int64_t per = ((int64_t)p.tiles_m * p.tiles_n + kNumXcd - 1) / kNumXcd;
  const int64_t most = L::kPerCu * kNumCu / kNumXcd;
  NE_CHECK_SUPPORTED(per < (int64_t(1) << 24), "too many tiles: %d x %d", p.tiles_m, p.tiles_n);
  const unsigned grid = (unsigned)((per < most ? per : most) * kNumXcd);
  hipLaunchKernelGGL((w8a8_tile_kernel<L, EPI>), dim3(grid), dim3(L::kWaves * kWave), 0, stream, p);
  return check_launch("w8a8_gemm");
}

// ---- few rows: fragments straight from memory ----------------------------------------
// Up to 64 rows a work-group's time is its round trips to memory, so nothing is staged: KG waves
// split k, load their fragments of 16 NS weight rows and all 16 PM token rows in the operand
// order (within a 128-byte line of k, lane group g takes bytes 32 g .. + 32, so that a row's
// line is read whole by four lanes), multiply, and the partial sums meet in LDS.  One row of 4,096 x
// 1,024: 3.5-3.7 us, 64 rows of 1,024 x 2,048: 4.9; the weights alone 0.8 and 0.4.
template <int PM_, int NS_, int KG_, int CG_>
struct FewLayout {
  static constexpr int PM = PM_, NS = NS_, KG = KG_, CG = CG_;  // CG column groups of 16 NS weight rows
  static constexpr int kWaves = KG * CG;
  static constexpr int kUnroll = PM >= 4 ? 2 : 4;  // 128-byte lines of k in flight
};

template <typename L, int EPI>
__global__ __launch_bounds__(L::kWaves* kWave) void w8a8_few_rows_kernel(W8a8Params p) {
  constexpr int PM = L::PM, NS = L::NS, KG = L::KG, CG = L::CG, U = L::kUnroll;
  __shared__ intx4 part[KG][CG][PM][NS][kWave];
  const int lane = threadIdx.x % kWave;
  const int r = lane & 15;
  const int g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kg = wave % KG, cg = wave / KG;
  const int n0 = (blockIdx.x * CG + cg) * 16 * NS;
  const int m0 = blockIdx.y * 16 * PM;
  const int k_chunks = p.k / 16;
  const int lines = (k_chunks + 7) / 8;
  const int8_t* wrow[NS];
  const int8_t* xrow[PM];
#pragma unroll
  for (int ns = 0; ns < NS; ++ns) wrow[ns] = p.w + (int64_t)min(n0 + ns * 16 + r, p.n - 1) * p.k + 32 * g;
#pragma unroll
  for (int mi = 0; mi < PM; ++mi) xrow[mi] = p.x + (int64_t)min(m0 + mi * 16 + r, p.m - 1) * p.ldx + 32 * g;
  intx4 acc[PM][NS];
#pragma unroll
  for (int mi = 0; mi < PM; ++mi)
#pragma unroll
    for (int ns = 0; ns < NS; ++ns) acc[mi][ns] = intx4{0, 0, 0, 0};
  for (int line0 = kg; line0 < lines; line0 += KG * U) {
    intx4 wf[U][2][NS], xf[U][2][PM];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int line = line0 + u * KG;
        const bool in = line * 8 + 2 * g + q < k_chunks;
        const int64_t at = (int64_t)line * 128 + 16 * q;
#pragma unroll
        for (int ns = 0; ns < NS; ++ns) wf[u][q][ns] = in ? *(const intx4*)(wrow[ns] + at) : intx4{0, 0, 0, 0};
#pragma unroll
        for (int mi = 0; mi < PM; ++mi) xf[u][q][mi] = in ? *(const intx4*)(xrow[mi] + at) : intx4{0, 0, 0, 0};
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int mi = 0; mi < PM; ++mi)
#pragma unroll
          for (int ns = 0; ns < NS; ++ns)
            acc[mi][ns] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][q][ns], xf[u][q][mi], acc[mi][ns], 0, 0, 0);
  }
  if constexpr (KG > 1) {
#pragma unroll
    for (int mi = 0; mi < PM; ++mi)
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) part[kg][cg][mi][ns][lane] = acc[mi][ns];
    __syncthreads();
  }
  // wave kg of a column group finishes the token subtiles kg, kg + KG, ..
  const int n_out = EPI == NE_EPILOGUE_SWIGLU ? p.n / 2 : p.n;
  const bool wide = (uintptr_t)p.y % 8 == 0 && p.ldy % 4 == 0;
#pragma unroll
  for (int mi = 0; mi < PM; ++mi) {
    if (mi % KG != kg) continue;
    intx4 sum[NS];
#pragma unroll
    for (int ns = 0; ns < NS; ++ns) {
      if constexpr (KG == 1) {
        sum[ns] = acc[mi][ns];
      } else {
        sum[ns] = part[0][cg][mi][ns][lane];
#pragma unroll
        for (int o = 1; o < KG; ++o) sum[ns] += part[o][cg][mi][ns][lane];
      }
    }
    const int m = m0 + mi * 16 + r;
    const float s = p.xs[min(m, p.m - 1)];
    float sc[NS][4];
#pragma unroll
    for (int ns = 0; ns < NS; ++ns)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[ns][i] = weight_scale(p, min(n0 + ns * 16 + 4 * g + i, p.n - 1));
    uint16_t* row = p.y + (int64_t)m * p.ldy;
    if (m >= p.m) continue;
    if constexpr (EPI == NE_EPILOGUE_SWIGLU) {
      static_assert(NS % 2 == 0, "gate and up subtiles in pairs");
#pragma unroll
      for (int o = 0; o < NS / 2; ++o)
        store_columns<2>(row, n0 / 2 + o * 16 + 4 * g, n_out, wide, swiglu4(sum[2 * o], sum[2 * o + 1], s, sc[2 * o], sc[2 * o + 1]));
    } else {
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) store_columns<2>(row, n0 + ns * 16 + 4 * g, n_out, wide, store4(sum[ns], s, sc[ns]));
    }
  }
}

template <typename L, int EPI>
int launch_few(const W8a8Params& p, hipStream_t stream) {
  const dim3 grid(ceil_div(p.n, 16 * L::NS * L::CG), ceil_div(p.m, 16 * L::PM));
  hipLaunchKernelGGL((w8a8_few_rows_kernel<L, EPI>), grid, dim3(L::kWaves * kWave), 0, stream, p);
  return check_launch("w8a8_gemm");
}

// ---- which kernel --------------------------------------------------------------------
// The least estimated time (us) over the kernels: a fixed part, and a cost per 128 k that grows
// with the tiles (or work-groups) per CU.  Constants fitted to 192 shapes (m 1-4,096, n 256-16,384,
// k 256-8,192, GPU time from graphs), over which the choice takes 1.5 % longer than the fastest
// kernel of each shape on average, at most 32 % (200 rows, n = 16,384, k = 8,192: 71 against 54 us).
// Examples (us; few rows / 64 x 64 / 64 x 128 / 128 x 128 / 256 x 256): 64 x 1,024 x 2,048 5.3 / 10.0 /
// 12.1 / 15.0 / 27.8, 333 x 4,096 x 1,024 14.4 / 8.8 / 8.7 / 10.1 / 18.8, 2,048 x 4,096 x 1,024 - / 21.3 /
// 19.4 / 16.0 / 21.9, 4,096 x 4,096 x 1,024 - / 37.6 / 32.1 / 25.2 / 23.2.
struct Kernel {
  int id;       // as ne_w8a8_kernel names it
  int variant;  // of the few-rows kernel: token subtiles, and 10 for two weight subtiles, 20 for two column groups
};

Kernel choose_kernel(int m, int n, int k, bool swiglu) {
  const double stages = (k + 127) / 128;
  Kernel best{};
  double least = 1e30;
  auto offer = [&](int id, int variant, double us) {
    if (us < least) {
      least = us;
      best = Kernel{id, variant};
    }
  };
  auto count = [&](int bm, int bn) { return (double)ceil_div(m, bm) * ceil_div(n, bn) / kNumCu; };
  auto tile = [&](int id, int bm, int bn, double fixed, double stage, double a, double b) {
    const double load = a + b * count(bm, bn);
    offer(id, 0, fixed + stage * stages * (load > 1 ? load : 1));
  };
  const double big = count(256, 256);
  offer(NE_W8A8_TILE_256X256, 0, 6.5 + 1.31 * stages * (big <= 0.125 ? 1 : 1.55 * ceil(big)));
  tile(NE_W8A8_TILE_128X128, 128, 128, 4.2, 0.69, 0.5, 0.85);
  tile(NE_W8A8_TILE_64X128, 64, 128, 4.0, 0.51, 0.25, 0.83);
  tile(NE_W8A8_TILE_64X64, 64, 64, 3.7, 0.39, 0.35, 0.62);
  auto few = [&](int variant, int rows, int columns, double line) {
    offer(NE_W8A8_FEW_ROWS, variant, 3.5 + line * stages * ceil(count(rows, columns)));
  };
  if (!swiglu) {
    few(1, 16, 16, 0.108);
    few(2, 32, 16, 0.16);
    few(4, 64, 16, 0.27);
    if (m <= 16) {
      const double load = count(16, 32);
      offer(NE_W8A8_FEW_ROWS, 21, 4.0 + 0.16 * stages * (load > 1 ? load : 1));
    }
  } else {
    few(11, 16, 32, 0.16);
    few(12, 32, 32, 0.22);
  }
  few(14, 64, 32, 0.34);
  return best;
}

template <int EPI>
int launch_kernel(const W8a8Params& p, hipStream_t stream) {
  constexpr bool kSwiglu = EPI == NE_EPILOGUE_SWIGLU;
  const Kernel kernel = choose_kernel(p.m, p.n, p.k, kSwiglu);
  switch (kernel.id) {
    case NE_W8A8_TILE_256X256: return launch_tile<TileLayout<256, 256, 4, 2, 2>, EPI>(p, stream);
    case NE_W8A8_TILE_128X128: return launch_tile<TileLayout<128, 128, 2, 2, 2>, EPI>(p, stream);
    case NE_W8A8_TILE_64X128: return launch_tile<TileLayout<64, 128, 2, 2, 3>, EPI>(p, stream);
    case NE_W8A8_TILE_64X64:  // (gate and up subtiles in one wave)
      return launch_tile<TileLayout<64, 64, kSwiglu ? 4 : 2, kSwiglu ? 1 : 2, 3>, EPI>(p, stream);
    default: break;
  }
  if constexpr (kSwiglu) {
    if (kernel.variant == 11) return launch_few<FewLayout<1, 2, 8, 1>, EPI>(p, stream);
    if (kernel.variant == 12) return launch_few<FewLayout<2, 2, 8, 1>, EPI>(p, stream);
  } else {
    if (kernel.variant == 1) return launch_few<FewLayout<1, 1, 8, 1>, EPI>(p, stream);
    if (kernel.variant == 2) return launch_few<FewLayout<2, 1, 8, 1>, EPI>(p, stream);
    if (kernel.variant == 4) return launch_few<FewLayout<4, 1, 8, 1>, EPI>(p, stream);
    if (kernel.variant == 21) return launch_few<FewLayout<1, 1, 4, 2>, EPI>(p, stream);
  }
  return launch_few<FewLayout<4, 2, 8, 1>, EPI>(p, stream);
}

// A wave's tile has a head's 128 columns, so that a vector's sum and largest value are four lanes' work and
// its RoPE pairs one lane's.  256 x 256 tiles where their last round over the CUs is nearly full (92 %: a rule
// fitted to the shape below alone, and off by about 1 us there at 3,000 rows with a bf16 cache, 30.2 / 29.0, and
// at 4,096 with an int8 one), else 128 x 128, two per CU (us, 16 + 8 heads, k = 1,024, int8 cache, 256 / 128; ne_w8a8_gemm into memory; the
// W8A16 product with the same epilogue): 512 rows 30.6 / 15.2; 8.8; 17.7, 2,048 31.8 / 19.2; 14.8; 32.0,
// 4,096 33.4 / 32.4; 21.8; 53.0 (bf16 cache 30.1 / 32.5), 6,000 55.9 / 48.1; 32.9; 80.4, 8,192 57.2 /
// 58.3; 37.1; 91.1 (bf16 52.8 / 60.2), 16,384 107 / 111; 68; 171.  The row kernel alone takes 68-71 at 8,192.
// What the epilogue adds is its arithmetic, ~500 vector operations per 16 rows of a head.
template <int EPI>
int launch_qkv(const W8a8QkvParams& p, hipStream_t stream) {
  const int64_t tiles = (int64_t)ceil_div(p.m, 256) * ceil_div(p.n, 256);
  if (tiles * 100 >= (tiles + kNumCu - 1) / kNumCu * kNumCu * 92)
    return launch_tile<TileLayout<256, 256, 4, 2, 2>, EPI>(p, stream);
  return launch_tile<TileLayout<128, 128, 4, 1, 2>, EPI>(p, stream);
}

}  // namespace

}  // namespace ne

using namespace ne;

namespace {

// what both products refuse
int check_product(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, const void* w_scale,
                  int32_t scale_dtype, int32_t m, int32_t n, int32_t k) {
  NE_CHECK_ARG(m >= 0 && n > 0 && k > 0, "bad gemm shape m=%d n=%d k=%d", m, n, k);
  NE_CHECK_SUPPORTED(k % 16 == 0 && k <= 131056, "k must be a multiple of 16 and at most 131,056 (got %d)", k);
  NE_CHECK_ARG(scale_dtype == NE_DTYPE_BF16 || scale_dtype == NE_DTYPE_FP16 || scale_dtype == NE_DTYPE_FP32,
               "scale_dtype must be bf16, fp16 or fp32");
  NE_CHECK_SUPPORTED(m <= (1 << 30) && n <= (1 << 30), "m and n must be at most 2^30 (got %d, %d)", m, n);
  if (m == 0) return NE_OK;
  NE_CHECK_ARG(x && x_scale && w && w_scale, "null pointer argument");
  NE_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldx < (1 << 23), "ldx must be >= k, a multiple of 16 and below 2^23 (got %lld)",
               (long long)ldx);
  NE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0, "x and w must be 16-byte aligned");
  NE_CHECK_ARG((uintptr_t)x_scale % 4 == 0 && (uintptr_t)w_scale % (scale_dtype == NE_DTYPE_FP32 ? 4 : 2) == 0,
               "scales off their type's alignment");
  return NE_OK;
}

}  // namespace

extern "C" int32_t ne_w8a8_kernel(int32_t m, int32_t n, int32_t k, int32_t epilogue) {
  if (m <= 0 || n <= 0 || k <= 0) return NE_W8A8_FEW_ROWS;
  return choose_kernel(m, n, k, epilogue == NE_EPILOGUE_SWIGLU).id;
}

extern "C" int ne_w8a8_gemm(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, const void* w_scale,
                            int32_t scale_dtype, int32_t m, int32_t n, int32_t k, void* y, int64_t ldy, int32_t epilogue,
                            void* stream) {
  NE_CHECK_ARG(epilogue == NE_EPILOGUE_STORE || epilogue == NE_EPILOGUE_SWIGLU, "unknown epilogue %d", epilogue);
  const int rc = check_product(x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k);
  if (rc != NE_OK) return rc;
  NE_CHECK_SUPPORTED(epilogue == NE_EPILOGUE_STORE || n % 32 == 0, "paired gate and up rows come in groups of 32 (n=%d)", n);
  if (m == 0) return NE_OK;
  NE_CHECK_ARG(y && (uintptr_t)y % 2 == 0, "null y, or off its type's alignment");
  NE_CHECK_ARG(ldy >= (epilogue == NE_EPILOGUE_SWIGLU ? n / 2 : n), "ldy too small (%lld)", (long long)ldy);
  const W8a8Params p{x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k, (uint16_t*)y, ldy, 0, 0};
  return epilogue == NE_EPILOGUE_SWIGLU ? launch_kernel<NE_EPILOGUE_SWIGLU>(p, (hipStream_t)stream)
                                        : launch_kernel<NE_EPILOGUE_STORE>(p, (hipStream_t)stream);
}

extern "C" int ne_w8a8_qkv_norm_rope_kv(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w,
                                        const void* w_scale, int32_t scale_dtype, int32_t m, int32_t num_q_heads,
                                        int32_t num_kv_heads, int32_t k, const void* q_norm_w, const void* k_norm_w, float eps,
                                        const int32_t* positions, const void* rope, int32_t rope_positions,
                                        const int32_t* slot_mapping, int32_t kv_dtype, void* k_cache, void* v_cache,
                                        void* k_scale, void* v_scale, int32_t kv_scale_dtype, void* q_out, void* stream) {
  NE_CHECK_ARG(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads <= (1 << 20) && num_kv_heads <= (1 << 20),
               "bad heads: %d and %d", num_q_heads, num_kv_heads);
  const int32_t n = (num_q_heads + 2 * num_kv_heads) * 128;
  const int rc = check_product(x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k);
  if (rc != NE_OK) return rc;
  NE_CHECK_ARG(kv_dtype == NE_DTYPE_BF16 || kv_dtype == NE_DTYPE_INT8, "kv_dtype must be int8 or bf16");
  const bool int8 = kv_dtype == NE_DTYPE_INT8;
  NE_CHECK_SUPPORTED(!int8 || kv_scale_dtype == NE_DTYPE_BF16 || kv_scale_dtype == NE_DTYPE_FP16,
                     "fused KV write supports bf16 or fp16 scales");
  NE_CHECK_ARG(rope_positions > 0, "rope_positions must be > 0");
  if (m == 0) return NE_OK;
  NE_CHECK_ARG(q_norm_w && k_norm_w && positions && rope && slot_mapping && k_cache && v_cache && q_out,
               "null pointer argument");
  NE_CHECK_ARG(!int8 || (k_scale && v_scale), "an int8 cache needs k_scale and v_scale");
  NE_CHECK_ARG((uintptr_t)q_out % 16 == 0 && (uintptr_t)k_cache % 16 == 0 && (uintptr_t)v_cache % 16 == 0,
               "q_out and the caches must be 16-byte aligned");
  NE_CHECK_ARG((uintptr_t)rope % 8 == 0 && (uintptr_t)q_norm_w % 4 == 0 && (uintptr_t)k_norm_w % 4 == 0,
               "rope must be 8-byte aligned, the norm weights 4-byte aligned");
  W8a8QkvParams p{};
  static_cast<W8a8Params&>(p) = W8a8Params{x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k, nullptr, 0, 0, 0};
  p.qkv = QkvRopeArgs{num_q_heads, num_kv_heads, (const uint16_t*)q_norm_w, (const uint16_t*)k_norm_w, eps, positions,
                      (const uint16_t*)rope, rope_positions, slot_mapping, k_cache, v_cache, k_scale, v_scale,
                      (uint16_t*)q_out, 0};
  p.kv_scale_dtype = kv_scale_dtype;
  return int8 ? launch_qkv<kEpilogueQkvInt8>(p, (hipStream_t)stream) : launch_qkv<kEpilogueQkvBf16>(p, (hipStream_t)stream);
}
