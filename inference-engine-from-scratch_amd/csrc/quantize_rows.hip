// Rows of activations to 8-bit integers with one scale per row, alone or in the RMSNorm that
// comes before a projection: what ne_w8a8_gemm multiplies.
//
//   s_i = max(max_j |x_ij|, 1e-8) / 127 in fp32,  q_ij = rint(x_ij / s_i)  (the formula of the
//   int8 cache and weights, ne/models/int8_quantization.py:30-34, per row of activations)
//
// The row maximum is taken over the bits of |x|, whose order is the values' with infinities and
// NaN above all: a row that holds one gets the scale NaN and codes 0, so that what it is
// multiplied into is NaN, as with the row itself.  Norm rows are the bits that ne_rmsnorm and
// ne_add_rmsnorm store (same sums in the same order, both roundings), quantised without the
// trip through memory.  Bound by memory where rows are many, each read once into registers (8,192 x
// 8,192 fp16 35-39 us, 5.2-5.8 TB/s; 4,001 x 2,048 8.6-8.9, of which ~2 are the launch; 8,192 x 1,024 through the
// norm 9.4, through add and norm 13.1, floors 4.9 and 11.5); few rows take a chain of one load, two
// reductions and a store (64 x 2,048 2.3-2.7 us replayed one after another, 64 x 1,024 through the norm 3.3, and
// up to 5.1 behind work that left the caches without them).
#include "ne_common.hpp"

namespace ne {

namespace {

enum { kPlain = 0, kNorm = 1, kAddNorm = 2 };

struct RowsParams {
  const uint16_t* x;  // plain and norm: the rows; add norm: delta
  int64_t ldx;
  uint16_t* residual;      // add norm: updated in place
  const uint16_t* weight;  // norm weight
  float eps;
  int8_t* codes;  // [rows][k]
  float* scales;  // [rows]
  int rows, k;
};

typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));

// the two values of a 32-bit word
template <int VDT>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (VDT == NE_DTYPE_BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    lo = f16_to_f32((uint16_t)(w & 0xFFFFu));
    hi = f16_to_f32((uint16_t)(w >> 16));
  }
}

template <int VDT>
__device__ __forceinline__ void unpack8(const u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2<VDT>(v[i], f[2 * i], f[2 * i + 1]);
}

__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}

// largest magnitude of 16-bit values, by their bits, in each half of `top`
__device__ __forceinline__ void max_magnitude(const u32x4 v, uint32_t& top) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, v[i] & 0x7FFF7FFFu),
                                                                 __builtin_bit_cast(ushort2v, top)));
}

// the larger half over the wave, in every lane
__device__ __forceinline__ uint32_t wave_max_half(uint32_t v) {
  v = max(v & 0xFFFFu, v >> 16);
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));   // quad_perm [1, 0, 3, 2]
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));   // quad_perm [2, 3, 0, 1]
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));  // row_half_mirror
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));  // row_mirror
  v = max(v, (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401F));               // lanes 16 apart
  return max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 32));
}

// the row's scale from the 16 bits of its largest magnitude; NaN where that is no number
template <int VDT>
__device__ __forceinline__ float row_scale(uint32_t top) {
  if (top >= (VDT == NE_DTYPE_BF16 ? 0x7F80u : 0x7C00u)) return __builtin_nanf("");
  const float v = VDT == NE_DTYPE_BF16 ? bf16_to_f32((uint16_t)top) : f16_to_f32((uint16_t)top);
  return fmaxf(v, 1e-8f) / 127.f;
}

// Codes of 8 values of a row with scale s, at most 127 in magnitude as no value exceeds the one the
// scale comes from (a row without a scale: 0).  One fma rounds x * v_rcp_f32(s) to a whole number
// in the low bits of 1.5 2^23; that product lies within 3e-5 of the fp32 quotient, so both round to the
// same number unless it is within 4e-5 of a half.  A wave with such a lane divides (one chunk
// of 512 values in 25).
template <int VDT>
__device__ __forceinline__ u32x2 quantize8(const u32x4 v, float s, float rcp) {
  constexpr float kWhole = 12582912.f;
  float f[8], t[8], far = 0.f;
  unpack8<VDT>(v, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    t[e] = __builtin_fmaf(f[e], rcp, kWhole);
    far = fmaxf(far, fabsf(__builtin_fmaf(f[e], rcp, -(t[e] - kWhole))));
  }
  if (__builtin_amdgcn_ballot_w64(far > 0.49996f) != 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = f[e] / s + kWhole;
  }
  u32x2 codes;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 1]), __float_as_uint(t[4 * i]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 3]), __float_as_uint(t[4 * i + 2]), 0x0c0c0400u);
    codes[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return s == s ? codes : u32x2{0, 0};
}

// WAVES waves per row (1: four rows per work-group; 4: one), CPL 8-element chunks per lane held in
// registers.  Every load of a row is issued before the first use.
template <int MODE, int VDT, int CPL, int WAVES>
__global__ __launch_bounds__(256) void quantize_rows_kernel(RowsParams p) {
  const int wave = threadIdx.x / kWave;
  const int row = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  if (WAVES == 1 && row >= p.rows) return;  // wave-uniform, and no barrier follows
  const int at = WAVES == 1 ? threadIdx.x % kWave : threadIdx.x;
  constexpr int kThreads = WAVES * kWave;
  const int chunks = p.k / 8;
  const uint16_t* src = p.x + (int64_t)row * p.ldx;
  u32x4 raw[CPL], wraw[CPL], draw[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ci = at + c * kThreads;
    raw[c] = u32x4{0, 0, 0, 0};
    if (ci < chunks) {
      if constexpr (MODE == kAddNorm) {
        raw[c] = *(const u32x4*)(p.residual + (int64_t)row * p.k + ci * 8);
        draw[c] = *(const u32x4*)(src + ci * 8);
      } else {
        raw[c] = *(const u32x4*)(src + ci * 8);
      }
      if constexpr (MODE != kPlain) wraw[c] = *(const u32x4*)(p.weight + ci * 8);
    }
  }
  uint32_t top = 0;
  if constexpr (MODE != kPlain) {
    // ne_rmsnorm's rows, by its operations in its order
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int ci = at + c * kThreads;
      if (ci < chunks) {
        float h[8];
        unpack8<VDT>(raw[c], h);
        if constexpr (MODE == kAddNorm) {
          float d[8];
          unpack8<VDT>(draw[c], d);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[e] += d[e];
          raw[c] = pack8(h);
          unpack8<VDT>(raw[c], h);
          *(u32x4*)(p.residual + (int64_t)row * p.k + ci * 8) = raw[c];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += h[e] * h[e];
      }
    }
    ss = wave_sum(ss);
    const float inv = rsqrtf(ss / (float)p.k + p.eps);
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int ci = at + c * kThreads;
      if (ci < chunks) {
        float h[8], w[8];
        unpack8<VDT>(raw[c], h);
        unpack8<VDT>(wraw[c], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] *= inv;
        unpack8<VDT>(pack8(h), h);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] *= w[e];
        raw[c] = pack8(h);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CPL; ++c) max_magnitude(raw[c], top);
  top = wave_max_half(top);
  if constexpr (WAVES > 1) {
    __shared__ uint32_t tops[WAVES];
    if (threadIdx.x % kWave == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, tops[w]);
  }
  const float s = row_scale<VDT>(top);
  if (at == 0) p.scales[row] = s;
  const float rcp = __builtin_amdgcn_rcpf(s);
  int8_t* dst = p.codes + (int64_t)row * p.k;
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int ci = at + c * kThreads;
    if (ci < chunks) *(u32x2*)(dst + ci * 8) = quantize8<VDT>(raw[c], s, rcp);
  }
}

// Rows too long for the registers: one work-group per row reads it twice (the second time from a cache).
template <int VDT>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(RowsParams p) {
  __shared__ uint32_t tops[16];
  const int row = blockIdx.x;
  const int chunks = p.k / 8;
  const uint16_t* src = p.x + (int64_t)row * p.ldx;
  uint32_t top = 0;
  for (int ci = threadIdx.x; ci < chunks; ci += 1024) max_magnitude(*(const u32x4*)(src + (int64_t)ci * 8), top);
  top = wave_max_half(top);
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) top = max(top, tops[w]);
  const float s = row_scale<VDT>(top);
  if (threadIdx.x == 0) p.scales[row] = s;
  const float rcp = __builtin_amdgcn_rcpf(s);
  int8_t* dst = p.codes + (int64_t)row * p.k;
  for (int ci = threadIdx.x; ci < chunks; ci += 1024)
    *(u32x2*)(dst + (int64_t)ci * 8) = quantize8<VDT>(*(const u32x4*)(src + (int64_t)ci * 8), s, rcp);
}

// Few waves per row leave a wave more to do, many take two rounds of the CUs.  us (bf16, replayed one after
// another on other rows each), one wave per row / four: 64 x 2,048 3.0 / 2.3, 320 x 2,048 3.5 / 3.0, 1,024 x
// 2,048 4.1 / 4.0, 4,001 x 2,048 8.9 / 8.8, 20,000 x 2,048 25.8 / 30.6; 64 x 4,096 4.3 / 2.6, 4,001 x 4,096 15.6 /
// 12.6, 20,000 x 4,096 50.8 / 45.6.  The norm's sum keeps ne_rmsnorm's order, one wave per row.
template <int MODE, int VDT>
int launch_rows(const RowsParams& p, hipStream_t stream) {
  const dim3 four(ceil_div(p.rows, 4)), one(p.rows), block(256);
  // a launch has fewer than 2^32 threads
  NE_CHECK_SUPPORTED(p.rows < (p.k <= (MODE == kPlain ? 2048 : 4096) ? 1 << 26 : p.k <= 16384 ? 1 << 24 : 1 << 22), "too many rows of %d: %d", p.k, p.rows);
#define NE_ROWS(CPL, WAVES, GRID) \
  hipLaunchKernelGGL((quantize_rows_kernel<MODE, VDT, CPL, WAVES>), GRID, block, 0, stream, p)
  if (p.k <= 512) {
    NE_ROWS(1, 1, four);
  } else if (p.k <= 1024) {
    NE_ROWS(2, 1, four);
  } else if constexpr (MODE == kPlain) {
    if (p.k <= 2048 && p.rows <= 2 * kNumCu) {
      NE_ROWS(1, 4, one);
    } else if (p.k <= 2048) {
      NE_ROWS(4, 1, four);
    } else if (p.k <= 4096) {
      NE_ROWS(2, 4, one);
    } else if (p.k <= 8192) {
      NE_ROWS(4, 4, one);
    } else if (p.k <= 16384) {
      NE_ROWS(8, 4, one);
    } else {
      hipLaunchKernelGGL(quantize_long_rows_kernel<VDT>, one, dim3(1024), 0, stream, p);
    }
  } else if (p.k <= 2048) {
    NE_ROWS(4, 1, four);
  } else {
    NE_ROWS(8, 1, four);
  }
#undef NE_ROWS
  return check_launch("quantize_rows");
}

constexpr int kMaxNormHidden = 4096;  // ne_rmsnorm's

int check_rows(const void* codes, const float* scales, int32_t rows, int32_t k) {
  NE_CHECK_ARG(rows >= 0 && k > 0, "bad shape: %d rows of %d", rows, k);
  NE_CHECK_SUPPORTED(k % 8 == 0, "rows must be a multiple of 8 wide (got %d)", k);
  if (rows == 0) return NE_OK;
  NE_CHECK_ARG(codes && scales, "null pointer argument");
  NE_CHECK_ARG((uintptr_t)codes % 8 == 0 && (uintptr_t)scales % 4 == 0, "codes must be 8-byte aligned, scales 4-byte aligned");
  return NE_OK;
}

int check_norm(const void* a, const void* b, const void* weight, int32_t k) {
  NE_CHECK_ARG(a && b && weight, "null pointer argument");
  NE_CHECK_SUPPORTED(k <= kMaxNormHidden, "hidden must be at most %d (got %d)", kMaxNormHidden, k);
  NE_CHECK_ARG((uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0 && (uintptr_t)weight % 16 == 0,
               "rows and weight must be 16-byte aligned");
  return NE_OK;
}

}  // namespace

}  // namespace ne

using namespace ne;

extern "C" int ne_quantize_rows(const void* x, int32_t dtype, int64_t ldx, int32_t rows, int32_t k, int8_t* codes,
                                float* scales, void* stream) {
  int rc = check_rows(codes, scales, rows, k);
  if (rc != NE_OK || rows == 0) return rc;
  NE_CHECK_ARG(x != nullptr, "null x");
  NE_CHECK_ARG(dtype == NE_DTYPE_BF16 || dtype == NE_DTYPE_FP16, "rows must be bf16 or fp16");
  NE_CHECK_ARG(ldx >= k && ldx % 8 == 0 && (uintptr_t)x % 16 == 0, "rows must be 16-byte aligned, ldx >= k");
  const RowsParams p{(const uint16_t*)x, ldx, nullptr, nullptr, 0.f, codes, scales, rows, k};
  return dtype == NE_DTYPE_BF16 ? launch_rows<kPlain, NE_DTYPE_BF16>(p, (hipStream_t)stream)
                                : launch_rows<kPlain, NE_DTYPE_FP16>(p, (hipStream_t)stream);
}

extern "C" int ne_rmsnorm_quantize(const void* x, const void* weight, int8_t* codes, float* scales, int32_t rows,
                                   int32_t hidden, float eps, void* stream) {
  int rc = check_rows(codes, scales, rows, hidden);
  if (rc != NE_OK || rows == 0) return rc;
  rc = check_norm(x, x, weight, hidden);
  if (rc != NE_OK) return rc;
  const RowsParams p{(const uint16_t*)x, hidden, nullptr, (const uint16_t*)weight, eps, codes, scales, rows, hidden};
  return launch_rows<kNorm, NE_DTYPE_BF16>(p, (hipStream_t)stream);
}

extern "C" int ne_add_rmsnorm_quantize(void* residual, const void* delta, const void* weight, int8_t* codes, float* scales,
                                       int32_t rows, int32_t hidden, float eps, void* stream) {
  int rc = check_rows(codes, scales, rows, hidden);
  if (rc != NE_OK || rows == 0) return rc;
  rc = check_norm(residual, delta, weight, hidden);
  if (rc != NE_OK) return rc;
  const RowsParams p{(const uint16_t*)delta, hidden, (uint16_t*)residual, (const uint16_t*)weight, eps, codes, scales, rows,
                     hidden};
  return launch_rows<kAddNorm, NE_DTYPE_BF16>(p, (hipStream_t)stream);
}
