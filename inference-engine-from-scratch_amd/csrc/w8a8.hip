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

// 16-byte source of the chunks past the end of k (a zero code adds nothing)
__device__ const u32x4 zero_chunk = {0, 0, 0, 0};

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
//   stage = 64 KS k of BM rows and BN weight rows, copied by DMA (global_load_lds_dwordx4), the
//           16-byte chunks of a row swizzled so that the fragment reads are free of bank conflicts
//   ring  = RING stages; a wave holds the next k-step's fragments while the MFMAs of the current
//           one run, and the barrier that admits a stage sits between two batches of MFMAs
template <int BM_, int BN_, int MW_, int NW_, int KS_, int RING_>
struct TileLayout {
  static constexpr int BM = BM_, BN = BN_, MW = MW_, NW = NW_, KS = KS_, RING = RING_;
  static constexpr int kWaves = MW * NW;
  static constexpr int PM = BM / MW / 16;   // token subtiles per wave
  static constexpr int NPW = BN / NW / 16;  // weight subtiles per wave
  static constexpr int kRow = 64 * KS;      // bytes of a row in a stage
  static constexpr int kStage = (BM + BN) * kRow;
  static constexpr int kCopies = kStage / 1024 / kWaves;  // per wave and stage
  static constexpr int kXCopies = BM * kRow / 1024 / kWaves;
  static constexpr int kLds = RING * kStage;
  static_assert(KS == 1 || KS == 2, "k-steps per stage");
  static_assert(BM * kRow % (1024 * kWaves) == 0 && BN * kRow % (1024 * kWaves) == 0, "copies split evenly over the waves");
  static_assert(RING >= 2 && kCopies * (RING - 1) < 64 && kLds <= 160 * 1024, "ring");
};

template <typename L, int EPI>
__global__ __launch_bounds__(L::kWaves* kWave) void w8a8_tile_kernel(W8a8Params p) {
  constexpr int PM = L::PM, NPW = L::NPW, KS = L::KS, RING = L::RING, D = L::kCopies;
  constexpr int kChunks = L::kRow / 16;      // per row
  constexpr int kCopyRows = 1024 / L::kRow;  // rows per copy
  __shared__ __attribute__((aligned(16))) char smem[L::kLds];
  // Each XCD takes a contiguous eighth of the tiles, in an order that walks all weight
  // tiles against groups of four row tiles: the group's rows stay in that XCD's L2.
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
  const int64_t per = (total + kNumXcd - 1) / kNumXcd;
  const int64_t idx = (int64_t)(blockIdx.x % kNumXcd) * per + blockIdx.x / kNumXcd;
  if (idx >= total) return;
  constexpr int kGroup = 4;
  const int grp = (int)(idx / ((int64_t)kGroup * p.tiles_n));
  const int in_grp = (int)(idx - (int64_t)grp * kGroup * p.tiles_n);
  const int rows_in = min(kGroup, p.tiles_m - grp * kGroup);
  const int tn = in_grp / rows_in;
  const int m0 = (grp * kGroup + in_grp - tn * rows_in) * L::BM;
  const int n0 = tn * L::BN;
  const int lane = threadIdx.x % kWave;
  const int r = lane & 15;
  const int g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int mw = wave / L::NW, nw = wave % L::NW;
  auto swizzle = [](int row) { return KS == 1 ? (row >> 1) & 3 : row & 7; };

  // Copy j of this wave is KiB j kWaves + wave of the stage: token rows, then weight rows.  Rows
  // past m and n re-read the last one and are never stored.
  const char* xbase = (const char*)p.x + (int64_t)m0 * p.ldx;
  const char* wbase = (const char*)p.w + (int64_t)n0 * p.k;
  uint32_t off[D];
  auto chunk_of = [&](int j) {
    const int row = (j * L::kWaves + wave) * kCopyRows + lane / kChunks - (j < L::kXCopies ? 0 : L::BM);
    return (lane % kChunks) ^ swizzle(row);
  };
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int row = (j * L::kWaves + wave) * kCopyRows + lane / kChunks;
    if (j < L::kXCopies) {
      off[j] = (uint32_t)min(row, p.m - 1 - m0) * (uint32_t)p.ldx + (uint32_t)(chunk_of(j) * 16);
    } else {
      off[j] = (uint32_t)min(row - L::BM, p.n - 1 - n0) * (uint32_t)p.k + (uint32_t)(chunk_of(j) * 16);
    }
  }
  const int n_stages = (p.k + L::kRow - 1) / L::kRow;
  const int k_chunks = p.k / 16;
  auto issue = [&](int t) {
    char* slot = smem + (t % RING) * L::kStage;
    const char* xs = uniform_ptr(xbase + (int64_t)t * L::kRow);
    const char* ws = uniform_ptr(wbase + (int64_t)t * L::kRow);
    if ((t + 1) * kChunks <= k_chunks) {
#pragma unroll
      for (int j = 0; j < D; ++j) {
        uint32_t o = off[j];
        __asm__("" : "+v"(o));  // keep the lane offset 32-bit: scalar base + offset addressing
        lds_dma16((j < L::kXCopies ? xs : ws) + o, slot + (j * L::kWaves + wave) * 1024);
      }
    } else {  // the last stage of a k off the stage's grid
#pragma unroll
      for (int j = 0; j < D; ++j) {
        const char* src = (j < L::kXCopies ? xs : ws) + off[j];
        if (t * kChunks + chunk_of(j) >= k_chunks) src = (const char*)&zero_chunk;
        lds_dma16(src, slot + (j * L::kWaves + wave) * 1024);
      }
    }
  };

  intx4 acc[PM][NPW];
#pragma unroll
  for (int mi = 0; mi < PM; ++mi)
#pragma unroll
    for (int ns = 0; ns < NPW; ++ns) acc[mi][ns] = intx4{0, 0, 0, 0};
  struct Frags {
    intx4 x[PM], w[NPW];
  };
  // chunk 4 q + g of a row sits at position chunk ^ swizzle(row); rows 16 apart swizzle alike
  auto read = [&](int t, int q, Frags& f) {
    const char* slot = smem + (t % RING) * L::kStage + (((4 * q + g) ^ swizzle(r)) * 16 + r * L::kRow);
#pragma unroll
    for (int ns = 0; ns < NPW; ++ns) f.w[ns] = *(const intx4*)(slot + (L::BM + (nw * NPW + ns) * 16) * L::kRow);
#pragma unroll
    for (int mi = 0; mi < PM; ++mi) f.x[mi] = *(const intx4*)(slot + (mw * PM + mi) * 16 * L::kRow);
  };
  auto mma = [&](const Frags& f, int from, int to) {
#pragma unroll
    for (int mi = 0; mi < PM; ++mi)
      if (mi >= from && mi < to) {
#pragma unroll
        for (int ns = 0; ns < NPW; ++ns)
          acc[mi][ns] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[ns], f.x[mi], acc[mi][ns], 0, 0, 0);
      }
  };
  // stage t + 1 has landed and every wave has read all of stage t: its slot takes stage t + RING
  auto advance = [&](int t) {
    wait_pending<D, RING - 2>(min(n_stages - 1, t + RING - 1) - (t + 1));
    wait_lgkmcnt0();
    asm volatile("s_barrier" ::: "memory");
    if (t + RING < n_stages) issue(t + RING);
  };

#pragma unroll
  for (int s = 0; s < RING; ++s)
    if (s < n_stages) issue(s);
  wait_pending<D, RING - 1>(min(n_stages, RING) - 1);  // stage 0 has landed
  asm volatile("s_barrier" ::: "memory");

  Frags a, b;
  read(0, 0, a);
  if constexpr (KS == 2) {
    for (int t = 0; t + 1 < n_stages; ++t) {
      read(t, 1, b);
      __builtin_amdgcn_sched_barrier(0);  // the reads go out before the multiplies
      mma(a, 0, PM);
      __builtin_amdgcn_sched_barrier(0);
      advance(t);
      read(t + 1, 0, a);
      __builtin_amdgcn_sched_barrier(0);
      mma(b, 0, PM);
      __builtin_amdgcn_sched_barrier(0);
    }
    read(n_stages - 1, 1, b);
    mma(a, 0, PM);
    mma(b, 0, PM);
  } else {
    auto step = [&](int t, Frags& cur, Frags& next) {
      mma(cur, 0, PM / 2);
      __builtin_amdgcn_sched_barrier(0);
      advance(t);
      read(t + 1, 0, next);
      __builtin_amdgcn_sched_barrier(0);
      mma(cur, PM / 2, PM);
      __builtin_amdgcn_sched_barrier(0);
    };
    int t = 0;
    for (; t + 2 < n_stages; t += 2) {
      step(t, a, b);
      step(t + 1, b, a);
    }
    if (t + 1 < n_stages) {
      step(t, a, b);
      mma(b, 0, PM);
    } else {
      mma(a, 0, PM);
    }
  }

  // lane (r, g): rows 16 mi + r, columns 16 ns + 4 g + i
  float sc[NPW][4], sx[PM];
#pragma unroll
  for (int ns = 0; ns < NPW; ++ns)
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[ns][i] = weight_scale(p, min(n0 + (nw * NPW + ns) * 16 + 4 * g + i, p.n - 1));
#pragma unroll
  for (int mi = 0; mi < PM; ++mi) sx[mi] = p.xs[min(m0 + (mw * PM + mi) * 16 + r, p.m - 1)];
  constexpr int kOut = EPI == NE_EPILOGUE_SWIGLU ? NPW / 2 : NPW;
  const int n_out = EPI == NE_EPILOGUE_SWIGLU ? p.n / 2 : p.n;
  const int col0 = (EPI == NE_EPILOGUE_SWIGLU ? n0 / 2 : n0) + nw * kOut * 16;
  const bool wide = (uintptr_t)p.y % 16 == 0 && p.ldy % 8 == 0;
#pragma unroll
  for (int mi = 0; mi < PM; ++mi) {
    const int m = m0 + (mw * PM + mi) * 16 + r;
    uint16_t* row = p.y + (int64_t)m * p.ldy;
    auto out4 = [&](int o) {
      if constexpr (EPI == NE_EPILOGUE_SWIGLU)
        return swiglu4(acc[mi][2 * o], acc[mi][2 * o + 1], sx[mi], sc[2 * o], sc[2 * o + 1]);
      return store4(acc[mi][o], sx[mi], sc[o]);
    };
    if constexpr (kOut % 2 == 0) {
#pragma unroll
      for (int o = 0; o < kOut; o += 2) {
        const u32x4 both = pair_columns(out4(o), out4(o + 1));
        if (m < p.m) store_columns<4>(row, col0 + o * 16 + pair_column(g), n_out, wide, both);
      }
    } else {
#pragma unroll
      for (int o = 0; o < kOut; ++o) {
        const u32x2 v = out4(o);
        if (m < p.m) store_columns<2>(row, col0 + o * 16 + 4 * g, n_out, wide, v);
      }
    }
  }
}

template <typename L, int EPI>
int launch_tile(W8a8Params p, hipStream_t stream) {
  p.tiles_m = ceil_div(p.m, L::BM);
  p.tiles_n = ceil_div(p.n, L::BN);
  const int64_t per = ((int64_t)p.tiles_m * p.tiles_n + kNumXcd - 1) / kNumXcd;
  NE_CHECK_SUPPORTED(per * kNumXcd < (int64_t(1) << 31) / 1024, "too many tiles: %d x %d", p.tiles_m, p.tiles_n);
  hipLaunchKernelGGL((w8a8_tile_kernel<L, EPI>), dim3((unsigned)(per * kNumXcd)), dim3(L::kWaves * kWave), 0, stream, p);
  return check_launch("w8a8_gemm");
}

// ---- few rows: fragments straight from memory ----------------------------------------
// Up to 64 rows a work-group's time is its round trips to memory, so nothing is staged: KG waves
// split k, load their fragments of 16 NS weight rows and all 16 PM token rows in the operand
// order (within a 128-byte line of k, lane group g takes bytes 32 g .. + 32, so that a row's
// line is read whole by four lanes), multiply, and the partial sums meet in LDS.
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

using Tile256x256 = TileLayout<256, 256, 2, 4, 1, 4>;
using Tile128x128 = TileLayout<128, 128, 2, 2, 1, 4>;
using Tile64x128 = TileLayout<64, 128, 1, 4, 1, 6>;

int32_t choose_kernel(int32_t m, int32_t n, int32_t k, bool swiglu) {
  if (m <= 64 && n <= 16384) return NE_W8A8_FEW_ROWS;
  const int64_t big = (int64_t)ceil_div(m, 256) * ceil_div(n, 256);
  if (big >= 128) return NE_W8A8_TILE_256X256;
  const int64_t mid = (int64_t)ceil_div(m, 128) * ceil_div(n, 128);
  return m > 64 && mid >= 128 ? NE_W8A8_TILE_128X128 : NE_W8A8_TILE_64X128;
}

template <int EPI>
int launch_kernel(int32_t kernel, const W8a8Params& p, hipStream_t stream) {
  constexpr int NS = EPI == NE_EPILOGUE_SWIGLU ? 2 : 1;
  switch (kernel) {
    case NE_W8A8_FEW_ROWS:
      if (p.m <= 16) return launch_few<FewLayout<1, NS, 8, 1>, EPI>(p, stream);
      if (p.m <= 32) return launch_few<FewLayout<2, NS, 8, 1>, EPI>(p, stream);
      return launch_few<FewLayout<4, NS, 8, 1>, EPI>(p, stream);
    case NE_W8A8_TILE_64X128: return launch_tile<Tile64x128, EPI>(p, stream);
    case NE_W8A8_TILE_128X128: return launch_tile<Tile128x128, EPI>(p, stream);
    default: return launch_tile<Tile256x256, EPI>(p, stream);
  }
}

}  // namespace

}  // namespace ne

using namespace ne;

extern "C" int32_t ne_w8a8_kernel(int32_t m, int32_t n, int32_t k, int32_t epilogue) {
  if (m <= 0 || n <= 0 || k <= 0) return NE_W8A8_FEW_ROWS;
  return choose_kernel(m, n, k, epilogue == NE_EPILOGUE_SWIGLU);
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
  if (m == 0) return NE_OK;
  NE_CHECK_ARG(x && x_scale && w && w_scale && y, "null pointer argument");
  NE_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldx < (1 << 23), "ldx must be >= k, a multiple of 16 and below 2^23 (got %lld)",
               (long long)ldx);
  NE_CHECK_ARG(ldy >= (epilogue == NE_EPILOGUE_SWIGLU ? n / 2 : n), "ldy too small (%lld)", (long long)ldy);
  NE_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0, "x and w must be 16-byte aligned");
  const W8a8Params p{x, ldx, x_scale, w, w_scale, scale_dtype, m, n, k, (uint16_t*)y, ldy, 0, 0};
  const int32_t kernel = choose_kernel(m, n, k, epilogue == NE_EPILOGUE_SWIGLU);
  return epilogue == NE_EPILOGUE_SWIGLU ? launch_kernel<NE_EPILOGUE_SWIGLU>(kernel, p, (hipStream_t)stream)
                                        : launch_kernel<NE_EPILOGUE_STORE>(kernel, p, (hipStream_t)stream);
}
