// Logits under penalties for repeated tokens, biases of single tokens and masks of allowed ones,
// before sampling or acceptance.  Per row, with c the token's occurrences in the row's output (the
// history after the prompt, and the guesses before the row in a verify step) and "seen" anywhere:
//   x1 = seen ? (x > 0 ? x / r : x r) : x     repetition
//   x2 = x1 - (f c + p [c > 0])               frequency and presence
//   x3 = x2 + bias,  x4 = allowed ? x3 : -inf
// in fp32, rounded once to the output's type.
//
// The counts need no state from step to step: they come from the history itself, which the
// caller holds anyway.  A work-group owns kRange tokens of one row, counts the history's tokens
// of its range in LDS (integer atomics: no order matters) while its logits are on their way to
// registers, and applies everything in one pass.  A word per token holds the output count in
// its low 31 bits and "in the prompt" in its top bit.  A history is read once per range (19 of
// 151,936 tokens), from the caches.
#include "ne_common.hpp"

namespace ne {

namespace {

struct AdjustParams {
  const void* logits;
  int64_t ld;
  void* out;
  int64_t ld_out;
  int rows, vocab;
  const int32_t* history;  // null: no penalties
  int64_t history_stride;
  const int32_t* history_len;
  const int32_t* prompt_len;  // null: 0
  int num_seqs, capacity;
  const int32_t* drafts;  // null: none
  int max_drafts;
  const int32_t* row_seq;     // null: row i is of sequence i
  const int32_t* row_drafts;  // null: 0
  const float *repetitions, *presences, *frequencies;
  float repetition, presence, frequency;
  const int32_t* bias_start;  // null: no biases
  const int32_t* bias_tokens;
  const float* bias_values;
  int num_biases;
  const uint8_t* allowed;  // null: every token
  int64_t allowed_stride;  // bytes
  const int32_t* allowed_rows;
  int num_allowed;
};

constexpr int kThreads = 512;
constexpr int kVectors = 2;                       // of 8 tokens per thread
constexpr int kRange = kThreads * kVectors * 8;   // tokens per work-group
constexpr uint32_t kInPrompt = 0x80000000u;

// eight values from any element's address (global loads need not be aligned)
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&f)[8]) {
  if constexpr (DT == NE_DTYPE_FP32) {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    const vec a = *(const vec*)((const float*)p + i), b = *(const vec*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = a[e];
      f[e + 4] = b[e];
    }
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
    const vec a = *(const vec*)((const uint16_t*)p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == NE_DTYPE_BF16) {
        f[2 * e] = __uint_as_float(a[e] << 16);
        f[2 * e + 1] = __uint_as_float(a[e] & 0xFFFF0000u);
      } else {
        f[2 * e] = f16_to_f32((uint16_t)(a[e] & 0xFFFFu));
        f[2 * e + 1] = f16_to_f32((uint16_t)(a[e] >> 16));
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&f)[8]) {
  if constexpr (DT == NE_DTYPE_FP32) {
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    *(vec*)((float*)p + i) = vec{f[0], f[1], f[2], f[3]};
    *(vec*)((float*)p + i + 4) = vec{f[4], f[5], f[6], f[7]};
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
    vec a;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == NE_DTYPE_BF16) {
        a[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
      } else {
        a[e] = (uint32_t)f32_to_f16(f[2 * e]) | (uint32_t)f32_to_f16(f[2 * e + 1]) << 16;
      }
    }
    *(vec*)((uint16_t*)p + i) = a;
  }
}

template <int IDT, int ODT>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(AdjustParams p) {
  extern __shared__ __attribute__((aligned(16))) uint32_t counts[];  // [kRange], then [kRange] bias entries + 1
  uint32_t* const entries = counts + (p.history ? kRange : 0);
  const int ranges = (p.vocab + kRange - 1) / kRange;
  const int row = blockIdx.x / ranges;
  const int base = (blockIdx.x - row * ranges) * kRange;
  const int tid = threadIdx.x;

  // which mask, and the bits of this thread's tokens
  uint32_t bits[kVectors];
  int mask = row;
  if (p.allowed && p.allowed_rows) mask = p.allowed_rows[row];
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int token = base + (v * kThreads + tid) * 8;
    bits[v] = 0xFFu;
    if (p.allowed && mask >= 0) bits[v] = mask < p.num_allowed && token < p.vocab ? p.allowed[mask * p.allowed_stride + token / 8] : 0u;
  }
  float x[kVectors][8];
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int token = base + (v * kThreads + tid) * 8;
    const int64_t at = (int64_t)row * p.ld + token;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[v][e] = 0.f;
    if (token + 8 <= p.vocab) {
      if (bits[v]) load8<IDT>(p.logits, at, x[v]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (token + e < p.vocab) x[v][e] = load_scale<IDT>(p.logits, at + e);
    }
  }

  const bool counted = p.history != nullptr, biased = p.bias_start != nullptr;
  if (counted || biased) {
    const int words = (counted && biased ? 2 : 1) * kRange;
    for (int i = tid * 4; i < words; i += kThreads * 4) *(u32x4*)(counts + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  if (counted) {
    const int seq = p.row_seq ? p.row_seq[row] : row;
    if (seq >= 0 && seq < p.num_seqs) {
      const int len = min(max(p.history_len[seq], 0), p.capacity);
      const int prompt = p.prompt_len ? p.prompt_len[seq] : 0;
      const int32_t* tokens = p.history + (int64_t)seq * p.history_stride;
      auto count = [&](int token, bool in_prompt) {
        const uint32_t u = (uint32_t)(token - base);
        if (u < (uint32_t)kRange && token < p.vocab) {
          if (in_prompt) {
            atomicOr(&counts[u], kInPrompt);
          } else {
            atomicAdd(&counts[u], 1u);
          }
        }
      };
      typedef int32_t vec __attribute__((ext_vector_type(4), aligned(4)));
      for (int i = tid * 4; i < len; i += kThreads * 4) {
        if (i + 4 <= len) {
          const vec t = *(const vec*)(tokens + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) count(t[e], i + e < prompt);
        } else {
          for (int e = i; e < len; ++e) count(tokens[e], e < prompt);
        }
      }
      if (p.drafts && p.row_drafts) {
        const int n = min(p.row_drafts[row], p.max_drafts);
        for (int i = tid; i < n; i += kThreads) count(p.drafts[(int64_t)seq * p.max_drafts + i], false);
      }
    }
  }
  if (biased) {  // of a token listed twice the last entry counts
    const int from = max(p.bias_start[row], 0), to = min(p.bias_start[row + 1], p.num_biases);
    for (int i = from + tid; i < to; i += kThreads) {
      const int token = p.bias_tokens[i];
      const uint32_t u = (uint32_t)(token - base);
      if (u < (uint32_t)kRange && token < p.vocab) atomicMax(&entries[u], (uint32_t)i + 1);
    }
  }
  if (counted || biased) __syncthreads();

  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (counted) {
    repetition = p.repetitions ? p.repetitions[row] : p.repetition;
    presence = p.presences ? p.presences[row] : p.presence;
    frequency = p.frequencies ? p.frequencies[row] : p.frequency;
    if (!(repetition > 0.f && repetition < __builtin_inff())) repetition = 1.f;
    if (presence != presence) presence = 0.f;
    if (frequency != frequency) frequency = 0.f;
  }
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int local = (v * kThreads + tid) * 8;
    const int token = base + local;
    if (token >= p.vocab) continue;
    if (counted) {
      const u32x4 a = *(const u32x4*)(counts + local), b = *(const u32x4*)(counts + local + 4);
      if ((a[0] | a[1] | a[2] | a[3] | b[0] | b[1] | b[2] | b[3]) != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t word = e < 4 ? a[e & 3] : b[e & 3];
          if (word != 0) {
            x[v][e] = x[v][e] > 0.f ? x[v][e] / repetition : x[v][e] * repetition;
            const uint32_t c = word & ~kInPrompt;
            if (c != 0) x[v][e] -= frequency * (float)c + presence;
          }
        }
      }
    }
    if (biased) {
      const u32x4 a = *(const u32x4*)(entries + local), b = *(const u32x4*)(entries + local + 4);
      if ((a[0] | a[1] | a[2] | a[3] | b[0] | b[1] | b[2] | b[3]) != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t entry = e < 4 ? a[e & 3] : b[e & 3];
          if (entry != 0) x[v][e] += p.bias_values[entry - 1];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!(bits[v] >> e & 1)) x[v][e] = -__builtin_inff();
    const int64_t at = (int64_t)row * p.ld_out + token;
    if (token + 8 <= p.vocab) {
      store8<ODT>(p.out, at, x[v]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (token + e < p.vocab) store_scale<ODT>(p.out, at + e, x[v][e]);
    }
  }
}

template <int IDT, int ODT>
int launch_adjust(const AdjustParams& p, hipStream_t stream) {
  const int64_t groups = (int64_t)p.rows * ceil_div(p.vocab, kRange);
  NE_CHECK_SUPPORTED(groups < (int64_t(1) << 31) / kThreads, "too many rows: %d of %d tokens", p.rows, p.vocab);
  const size_t lds = ((p.history ? 1 : 0) + (p.bias_start ? 1 : 0)) * kRange * sizeof(uint32_t);
  hipLaunchKernelGGL((adjust_logits_kernel<IDT, ODT>), dim3((unsigned)groups), dim3(kThreads), lds, stream, p);
  return check_launch("adjust_logits");
}

}  // namespace

}  // namespace ne

using namespace ne;

extern "C" int ne_adjust_logits(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t vocab,
                                const int32_t* history, int64_t history_stride, int32_t capacity,
                                const int32_t* history_len, const int32_t* prompt_len, int32_t num_seqs,
                                const int32_t* drafts, int32_t max_drafts, const int32_t* row_seq,
                                const int32_t* row_drafts, const float* repetitions, float repetition,
                                const float* presences, float presence, const float* frequencies, float frequency,
                                const int32_t* bias_start, const int32_t* bias_tokens, const float* bias_values,
                                int32_t num_biases, const int32_t* allowed, int64_t allowed_stride,
                                int32_t num_allowed, const int32_t* allowed_rows, void* out, int32_t out_dtype,
                                int64_t ld_out, void* stream) {
  NE_CHECK_ARG(rows >= 0 && vocab > 0, "bad shape: %d rows of %d", rows, vocab);
  NE_CHECK_SUPPORTED(vocab <= (1 << 24), "vocab must be at most 2^24 (got %d)", vocab);
  if (rows == 0) return NE_OK;
  NE_CHECK_ARG(logits && out, "null pointer argument");
  NE_CHECK_ARG(dtype == NE_DTYPE_BF16 || dtype == NE_DTYPE_FP16 || dtype == NE_DTYPE_FP32, "logits must be bf16, fp16 or fp32");
  NE_CHECK_ARG(out_dtype == dtype || out_dtype == NE_DTYPE_FP32, "out must be of the logits' type or fp32");
  NE_CHECK_ARG(ld >= vocab && ld_out >= vocab, "rows of %d tokens overlap (ld %lld, ld_out %lld)", vocab, (long long)ld,
               (long long)ld_out);
  const int64_t size = dtype == NE_DTYPE_FP32 ? 4 : 2, size_out = out_dtype == NE_DTYPE_FP32 ? 4 : 2;
  NE_CHECK_ARG((uintptr_t)logits % size == 0 && (uintptr_t)out % size_out == 0, "logits or out off their type's alignment");
  const char *a = (const char*)logits, *b = (const char*)out;
  const bool same = a == b && dtype == out_dtype && (ld == ld_out || rows == 1);
  NE_CHECK_ARG(same || a + ((int64_t)(rows - 1) * ld + vocab) * size <= b || b + ((int64_t)(rows - 1) * ld_out + vocab) * size_out <= a,
               "out overlaps the logits without being them");
  if (history) {
    NE_CHECK_ARG(history_len && num_seqs >= 0 && capacity >= 0 && capacity <= (1 << 30) && history_stride >= capacity,
                 "bad history: %d sequences of %d tokens, stride %lld", num_seqs, capacity, (long long)history_stride);
    NE_CHECK_ARG(row_seq || rows <= num_seqs, "%d rows of %d sequences need row_seq", rows, num_seqs);
    NE_CHECK_ARG(!drafts || (max_drafts >= 0 && row_drafts), "guesses need row_drafts");
    NE_CHECK_ARG(repetitions || (repetition > 0.f && repetition < __builtin_inff()), "repetition must be positive and finite");
    NE_CHECK_ARG((presences || presence == presence) && (frequencies || frequency == frequency),
                 "presence and frequency must not be NaN");
  }
  NE_CHECK_ARG(!bias_start || (num_biases >= 0 && (num_biases == 0 || (bias_tokens && bias_values))), "bad biases");
  if (allowed) {
    NE_CHECK_ARG(num_allowed >= 0 && allowed_stride >= (vocab + 31) / 32, "masks of %lld words for %d tokens",
                 (long long)allowed_stride, vocab);
    NE_CHECK_ARG(allowed_rows || rows <= num_allowed, "%d rows of %d masks need allowed_rows", rows, num_allowed);
  }
  const AdjustParams p{logits, ld, out, ld_out, rows, vocab, history, history_stride, history_len, prompt_len, num_seqs,
                       capacity, drafts, max_drafts, row_seq, row_drafts, repetitions, presences, frequencies, repetition,
                       presence, frequency, bias_start, bias_tokens, bias_values, num_biases, (const uint8_t*)allowed,
                       allowed_stride * 4, allowed_rows, num_allowed};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == NE_DTYPE_FP32) return launch_adjust<NE_DTYPE_FP32, NE_DTYPE_FP32>(p, s);
  if (dtype == NE_DTYPE_BF16)
    return out_dtype == NE_DTYPE_FP32 ? launch_adjust<NE_DTYPE_BF16, NE_DTYPE_FP32>(p, s)
                                      : launch_adjust<NE_DTYPE_BF16, NE_DTYPE_BF16>(p, s);
  return out_dtype == NE_DTYPE_FP32 ? launch_adjust<NE_DTYPE_FP16, NE_DTYPE_FP32>(p, s)
                                    : launch_adjust<NE_DTYPE_FP16, NE_DTYPE_FP16>(p, s);
}
