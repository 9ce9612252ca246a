// W8A8 products for gfx950: y[m, n] = bf16((sum_k q[m, k] w[n, k]) s[m] t[n]) for rows of 8-bit
// activations q with one scale each (quantize_rows.hip) and the int8 weights and row scales
// that the W8A16 products read.  The sum is exact in int32 (k <= 131,056 holds any codes), so
// no result depends on how k is split or ordered: every kernel here gives the same bits.
//
// As in gemm.hip an MFMA computes D = W . X^T (v_mfma_i32_16x16x64_i8), so that a lane holds
// four consecutive output columns of one token row.
#include "ne_common.hpp"

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

__device__ __forceinline__ void lds_dma16(const void* src, void* lds_wave_base) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
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
__global__ __launch_bounds__(L::kWaves* kWave) void w8a8_tile_kernel(W8a8Params p) {
  constexpr int PM = L::PM, NPW = L::NPW, RING = L::RING, D = L::kCopies;
  constexpr int kOut = EPI == NE_EPILOGUE_SWIGLU ? NPW / 2 : NPW;
  constexpr int kStores = PM * kOut / 2;  // of a wave's whole tile
  static_assert(D * (RING - 1) + kStores < 64, "vmcnt range");
  __shared__ __attribute__((aligned(16))) char smem[L::kLds];
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
      const int t = threadIdx.x;
      if (t < L::BM) return ((const uint32_t*)p.xs)[min(m0 + t, p.m - 1)];
      const int n = min(n0 + min(t - L::BM, L::BN - 1), p.n - 1);
      return p.ws_dtype == NE_DTYPE_FP32 ? ((const uint32_t*)p.ws)[n] : ((const uint16_t*)p.ws)[n];
    };
    auto put_scale = [&](uint32_t bits) {
      const bool fp32 = threadIdx.x < L::BM || p.ws_dtype == NE_DTYPE_FP32;
      const float half = p.ws_dtype == NE_DTYPE_BF16 ? bf16_to_f32((uint16_t)bits) : f16_to_f32((uint16_t)bits);
      const float v = fp32 ? __uint_as_float(bits) : half;
      if (L::BM + L::BN == L::kWaves * kWave || threadIdx.x < L::BM + L::BN) scales[threadIdx.x] = v;
    };
    uint32_t scale = 0;
#pragma unroll
    for (int mi = 0; mi < PM; ++mi)
#pragma unroll
      for (int ns = 0; ns < NPW; ++ns) acc[mi][ns] = intx4{0, 0, 0, 0};
    read(slot, 0, a);
#pragma unroll 1
    for (int t = 0; t < n_stages; ++t, ++s) {
      wait_lgkmcnt0();  // for a's reads, not for the next ones too
      read(slot, 1, b);
      if (t + 1 == n_stages) scale = my_scale();
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
    if (s - 1 + RING < all) issue();
    lds_barrier();

    // lane (r, g): rows 16 mi + r, columns 16 ns + 4 g + i
    int l = lane;
    __asm__ volatile("" : "+v"(l));  // addresses made here, not kept in registers through the k loop
    const int er = l & 15, eg = l >> 4;
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
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);  // the stores stay before the next wait
  }
}

template <typename L, int EPI>
int launch_tile(W8a8Params p, hipStream_t stream) {
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
// kernel of each shape on average, at most 30 % (200 rows, n = 16,384, k = 8,192: 71 against 54 us).
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

}  // namespace

}  // namespace ne

using namespace ne;

extern "C" int32_t ne_w8a8_kernel(int32_t m, int32_t n, int32_t k, int32_t epilogue) {
  if (m <= 0 || n <= 0 || k <= 0) return NE_W8A8_FEW_ROWS;
  return choose_kernel(m, n, k, epilogue == NE_EPILOGUE_SWIGLU).id;
}

extern "C" int ne_w8a8_gemm(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, const void* w_scale,
                            int32_t scale_dtype, int32_t m, int32_t n, int32_t k, void* y, int64_t ldy, int32_t epilogue,
                            void* stream) {
  NE_CHECK_ARG(m >= 0 && n > 0 && k > 0, "bad gemm shape m=%d n=%d k=%d", m, n, k);
  NE_CHECK_ARG(epilogue == NE_EPILOGUE_STORE || epilogue == NE_EPILOGUE_SWIGLU, "unknown epilogue %d", epilogue);
  NE_CHECK_SUPPORTED(k % 16 == 0 && k <= 131056, "k must be a multiple of 16 and at most 131,056 (got %d)", k);
  NE_CHECK_SUPPORTED(epilogue == NE_EPILOGUE_STORE || n % 32 == 0, "paired gate and up rows come in groups of 32 (n=%d)", n);
  NE_CHECK_ARG(scale_dtype == NE_DTYPE_BF16 || scale_dtype == NE_DTYPE_FP16 || scale_dtype == NE_DTYPE_FP32,
               "scale_dtype must be bf16, fp16 or fp32");
  NE_CHECK_SUPPORTED(m <= (1 << 30) && n <= (1 << 30), "m and n must be at most 2^30 (got %d, %d)", m, n);
  if (m == 0) return NE_OK;
  NE_CHECK_ARG(x && x_scale && w && w_scale && y, "null pointer argument");
  NE_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldx < (1 << 23), "ldx must be >= k, a multiple of 16 and below 2^23 (got %lld)",
               (long long)ldx);
  NE_CHECK_ARG(ldy >= (epilogue == NE_EPILOGUE_SWIGLU ? n / 2 : n), "ldy too small (%lld)", (long long)ldy);
  NE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0, "x and w must be 16-byte aligned");
  NE_CHECK_ARG((uintptr_t)x_scale % 4 == 0 && (uintptr_t)w_scale % (scale_dtype == NE_DTYPE_FP32 ? 4 : 2) == 0 && (uintptr_t)y % 2 == 0,
               "scales or y off their type's alignment");
  const W8a8Params p{x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k, (uint16_t*)y, ldy, 0, 0};
  return epilogue == NE_EPILOGUE_SWIGLU ? launch_kernel<NE_EPILOGUE_SWIGLU>(p, (hipStream_t)stream)
                                        : launch_kernel<NE_EPILOGUE_STORE>(p, (hipStream_t)stream);
}
