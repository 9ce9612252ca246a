// What the paged attention kernels have in common (gfx950): element types and conversions,
// Q fragments, and the query-tile kernels' staging of 128 keys of one KV head into LDS as
// MFMA operands (K rows, V transposed, int8 codes converted once).
//
// Parameters P of the staging: k_cache, v_cache, k_scale, v_scale and num_kv_heads.
#pragma once

#include "ne_common.hpp"

namespace ne {

namespace {

constexpr int kHeadDim = 128;
constexpr int kRows = 16;       // MFMA M/N tile = query rows per unit
constexpr int kTileKeys = 16;   // keys per MFMA tile (never straddles a block)
constexpr float kNegBig = -1e30f;  // finite "minus infinity" for running maxima
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyMaxVScale = 128.f;  // P * scale <= 2^8 * 128 stays inside fp16

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// int8 codes -> fp16 (exact: |code| <= 127), one SDWA convert per value, built as a
// whole MFMA operand (4 dwords) per asm block.  The compiler sees no instruction
// inside an asm block, so it cannot insert the wait states CDNA needs between a
// VALU write of a VGPR and an MFMA reading it (two): every block ends with s_nop 1,
// which gives them to whichever instruction consumes the result.
#define NE_CVT_LO(D, S, B) "v_cvt_f16_i16_sdwa " D ", sext(" S ") dst_sel:WORD_0 dst_unused:UNUSED_PAD src0_sel:BYTE_" #B "\n\t"
#define NE_CVT_HI(D, S, B) "v_cvt_f16_i16_sdwa " D ", sext(" S ") dst_sel:WORD_1 dst_unused:UNUSED_PRESERVE src0_sel:BYTE_" #B "\n\t"

// K operand: bytes 0..3 of w0 then of w1, in order.
__device__ __forceinline__ u32x4 i8x8_f16x8(uint32_t w0, uint32_t w1) {
  uint32_t a, b, c, d;
  asm(NE_CVT_LO("%0", "%4", 0) NE_CVT_HI("%0", "%4", 1) NE_CVT_LO("%1", "%4", 2) NE_CVT_HI("%1", "%4", 3)
      NE_CVT_LO("%2", "%5", 0) NE_CVT_HI("%2", "%5", 1) NE_CVT_LO("%3", "%5", 2) NE_CVT_HI("%3", "%5", 3)
      "s_nop 1"
      : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d)
      : "v"(w0), "v"(w1));
  return u32x4{a, b, c, d};
}

// V^T operand: byte B of each of the eight key rows x[0..7], in key order.
#define NE_CVT_COLS(B)                                                                          \
  asm(NE_CVT_LO("%0", "%4", B) NE_CVT_HI("%0", "%5", B) NE_CVT_LO("%1", "%6", B)               \
          NE_CVT_HI("%1", "%7", B) NE_CVT_LO("%2", "%8", B) NE_CVT_HI("%2", "%9", B)            \
              NE_CVT_LO("%3", "%10", B) NE_CVT_HI("%3", "%11", B) "s_nop 1"                     \
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])                                      \
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]))

template <int B>
__device__ __forceinline__ u32x4 i8_cols_f16x8(const uint32_t (&x)[8]) {
  uint32_t r[4];
  if constexpr (B == 0) {
    NE_CVT_COLS(0);
  } else if constexpr (B == 1) {
    NE_CVT_COLS(1);
  } else if constexpr (B == 2) {
    NE_CVT_COLS(2);
  } else {
    NE_CVT_COLS(3);
  }
  return u32x4{r[0], r[1], r[2], r[3]};
}
#undef NE_CVT_COLS
#undef NE_CVT_LO
#undef NE_CVT_HI

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  floatx2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Q fragments of the B operand: fp16 for the int8 cache (int8 codes are exact in
// fp16, so S keeps the bf16 product's value), bf16 otherwise.
template <bool INT8>
struct QFrag;
template <>
struct QFrag<true> {
  f16x8 q[4];
};
template <>
struct QFrag<false> {
  bf16x8 q[4];
};

constexpr int kQtWaves = 8;
constexpr int kQtKeys = 128;                     // keys per stage
constexpr int kQtMT = 2;                         // 16-row MFMA tiles per wave
constexpr int kQtWaveRows = kQtMT * kRows;
constexpr int kQtThreads = kQtWaves * kWave;
constexpr int kQtTileBytes = kQtKeys * kHeadDim * 2;  // one stage's K (or V^T), 16-bit
constexpr int kQtStage = 2 * kQtTileBytes;
constexpr int kQtScaleOff = 2 * kQtStage;        // float [2 buffers][K | V][128 keys]
constexpr int kQtSlotOff = kQtScaleOff + 2 * 2 * kQtKeys * 4;  // int [2][8 tiles]
constexpr int kQtFlagOff = kQtSlotOff + 2 * 8 * 4;             // int [2 buffers][2 waves]
constexpr int kQtScanOff = kQtFlagOff + 2 * 2 * 4;             // int [3][8 waves], [4]
constexpr int kQtLds = kQtScanOff + 28 * 4;
static_assert(kQtLds <= 160 * 1024, "LDS of one CU");

// One thread's share of a stage on its way to LDS.
template <bool INT8>
struct QtRegs;
template <>
struct QtRegs<true> {
  u32x4 k[2];     // keys tid / 8 + 64 j, codes 16 (tid % 8) .. + 16
  uint32_t v[8];  // the 8 keys of octet tid / 32, codes 4 (tid % 32) .. + 4
  float sc;       // thread < 128: key scale; < 256: value scale of key tid % 128
};
template <>
struct QtRegs<false> {
  u32x4 k[4];  // keys tid / 16 + 32 j, dims 8 (tid % 16) .. + 8
  u32x2 v[8];  // the 8 keys of octet tid / 32, dims 4 (tid % 32) .. + 4
};

// Key of octet o (0..15), element e: the contraction order of the second product, whose
// P operand holds keys 16 (e / 4) + 4 g + e % 4 of a 32-key step (o = 4 step + g).
__device__ __forceinline__ int qt_octet_key(int o, int e) {
  return 32 * (o >> 2) + 16 * (e >> 2) + 4 * (o & 3) + (e & 3);
}

// 16-byte chunk position in the LDS rows (256 B: a key's dims, or a dim's keys): spreads
// both the transposing writes (rows 4 apart) and the fragment reads (rows 1 apart)
__device__ __forceinline__ int qt_k_pos(int key, int chunk) { return chunk ^ (key & 15); }
__device__ __forceinline__ int qt_v_pos(int dim, int chunk) { return chunk ^ ((dim ^ ((dim >> 3) & 1)) & 7); }

template <bool INT8, int SDT, typename P>
__device__ __forceinline__ void qt_load(const P& p, const int* s_slot, int kb, int kend, int head,
                                        int tid, QtRegs<INT8>& R) {
  constexpr int kEsz = INT8 ? 1 : 2;
  const int64_t slot_bytes = (int64_t)p.num_kv_heads * kHeadDim * kEsz;
  const char* kc = (const char*)p.k_cache + (int64_t)head * kHeadDim * kEsz;
  const char* vc = (const char*)p.v_cache + (int64_t)head * kHeadDim * kEsz;
#pragma unroll
  for (int j = 0; j < (INT8 ? 2 : 4); ++j) {
    const int key = INT8 ? (tid >> 3) + 64 * j : (tid >> 4) + 32 * j;
    const int64_t slot = s_slot[key >> 4] + (key & 15);
    R.k[j] = *(const u32x4*)(kc + slot * slot_bytes + 16 * (tid & (INT8 ? 7 : 15)));
  }
  const int o = tid >> 5;
  const int64_t slot0 = s_slot[2 * (o >> 2)] + 4 * (o & 3);
  const int64_t slot1 = s_slot[2 * (o >> 2) + 1] + 4 * (o & 3);
  const char* v0 = vc + slot0 * slot_bytes + 4 * kEsz * (tid & 31);
  const char* v1 = vc + slot1 * slot_bytes + 4 * kEsz * (tid & 31);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const char* src = (e < 4 ? v0 : v1) + (e & 3) * slot_bytes;
    if constexpr (INT8) {
      R.v[e] = *(const uint32_t*)src;
    } else {
      R.v[e] = *(const u32x2*)src;
    }
  }
  if constexpr (INT8) {
    R.sc = 0.f;
    if (tid < 2 * kQtKeys) {  // whole waves
      const int key = tid & (kQtKeys - 1);
      const int64_t slot = s_slot[key >> 4] + (key & 15);
      const float s = load_scale<SDT>(tid < kQtKeys ? p.k_scale : p.v_scale, slot * p.num_kv_heads + head);
      R.sc = kb + key < kend ? s : 0.f;  // a slot past the context's end may hold anything
    }
  } else {
    // bf16 values past the context's end may be stale bit patterns: 0 * NaN must not
    // reach the product (int8 codes are always finite)
    if (kb + kQtKeys > kend) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (kb + qt_octet_key(o, e) >= kend) R.v[e] = u32x2{0, 0};
    }
  }
}

template <bool INT8>
__device__ __forceinline__ void qt_store_kv(char* smem, int buf, int tid, const QtRegs<INT8>& R) {
  char* ks = smem + buf * kQtStage;
  char* vs = ks + kQtTileBytes;
  const int o = tid >> 5;
  const int q = tid & 31;
  if constexpr (INT8) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = (tid >> 3) + 64 * j;
      const int c = 2 * (tid & 7);
      *(u32x4*)(ks + key * 256 + qt_k_pos(key, c) * 16) = i8x8_f16x8(R.k[j][0], R.k[j][1]);
      *(u32x4*)(ks + key * 256 + qt_k_pos(key, c + 1) * 16) = i8x8_f16x8(R.k[j][2], R.k[j][3]);
    }
    *(u32x4*)(vs + (4 * q + 0) * 256 + qt_v_pos(4 * q + 0, o) * 16) = i8_cols_f16x8<0>(R.v);
    *(u32x4*)(vs + (4 * q + 1) * 256 + qt_v_pos(4 * q + 1, o) * 16) = i8_cols_f16x8<1>(R.v);
    *(u32x4*)(vs + (4 * q + 2) * 256 + qt_v_pos(4 * q + 2, o) * 16) = i8_cols_f16x8<2>(R.v);
    *(u32x4*)(vs + (4 * q + 3) * 256 + qt_v_pos(4 * q + 3, o) * 16) = i8_cols_f16x8<3>(R.v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = (tid >> 4) + 32 * j;
      *(u32x4*)(ks + key * 256 + qt_k_pos(key, tid & 15) * 16) = R.k[j];
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int w = b >> 1;
      const uint32_t sel = (b & 1) ? 0x07060302u : 0x05040100u;
      const u32x4 col = {__builtin_amdgcn_perm(R.v[1][w], R.v[0][w], sel), __builtin_amdgcn_perm(R.v[3][w], R.v[2][w], sel),
                         __builtin_amdgcn_perm(R.v[5][w], R.v[4][w], sel), __builtin_amdgcn_perm(R.v[7][w], R.v[6][w], sel)};
      *(u32x4*)(vs + (4 * q + b) * 256 + qt_v_pos(4 * q + b, o) * 16) = col;
    }
  }
}

template <bool INT8>
__device__ __forceinline__ void qt_store(char* smem, int buf, int tid, int wave, int lane, float qk_scale,
                                         const QtRegs<INT8>& R) {
  qt_store_kv<INT8>(smem, buf, tid, R);
  if constexpr (INT8) {
    if (tid < 2 * kQtKeys) {
      // key scales carry the softmax scale; value scales the fp16 range check
      float* sc = (float*)(smem + kQtScaleOff) + buf * 2 * kQtKeys;
      sc[tid] = tid < kQtKeys ? R.sc * qk_scale : R.sc;
      const bool big = __ballot(R.sc > kLazyMaxVScale) != 0;
      if (tid >= kQtKeys && lane == 0) ((int*)(smem + kQtFlagOff))[buf * 2 + wave - kQtKeys / kWave] = big;
    }
  }
}

}  // namespace

}  // namespace ne
