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

using ConstF32 = __attribute__((address_space(4))) const float;  // as ConstI32
constexpr int kMaxNarrow = 32767;
constexpr int kRowsPerSlice = 32767;  // of the grid

// Eight values as they lie in memory, from any element's address (global accesses need not be
// aligned).
template <int DT>
struct Raw {
  static constexpr int kWords = DT == NE_DTYPE_FP32 ? 8 : 4;
  uint32_t word[kWords];
};

template <int DT>
__device__ __forceinline__ const void* element(const void* p, int64_t i) {
  return (const char*)p + i * (DT == NE_DTYPE_FP32 ? 4 : 2);
}

template <int DT>
__device__ __forceinline__ Raw<DT> load8(const void* p, int64_t i) {
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
  Raw<DT> r;
#pragma unroll
  for (int w = 0; w < Raw<DT>::kWords; w += 4) {
    const vec a = *(const vec*)((const char*)element<DT>(p, i) + w * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.word[w + e] = a[e];
  }
  return r;
}

template <int DT>
__device__ __forceinline__ float value_of(const Raw<DT>& r, int e) {
  if constexpr (DT == NE_DTYPE_FP32) return __uint_as_float(r.word[e]);
  const uint32_t half = e % 2 ? r.word[e / 2] >> 16 : r.word[e / 2] & 0xFFFFu;
  return DT == NE_DTYPE_BF16 ? bf16_to_f32((uint16_t)half) : f16_to_f32((uint16_t)half);
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&f)[8]) {
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
  uint32_t word[Raw<DT>::kWords];
#pragma unroll
  for (int w = 0; w < Raw<DT>::kWords; ++w) {
    if constexpr (DT == NE_DTYPE_FP32) {
      word[w] = __float_as_uint(f[w]);
    } else if constexpr (DT == NE_DTYPE_BF16) {
      word[w] = pack_bf16x2(f[2 * w], f[2 * w + 1]);
    } else {
      word[w] = (uint32_t)f32_to_f16(f[2 * w]) | (uint32_t)f32_to_f16(f[2 * w + 1]) << 16;
    }
  }
#pragma unroll
  for (int w = 0; w < Raw<DT>::kWords; w += 4)
    *(vec*)((char*)element<DT>(p, i) + w * 4) = vec{word[w], word[w + 1], word[w + 2], word[w + 3]};
}

// WIDE: a 32-bit word per token; otherwise 16 bits (histories of at most kMaxNarrow tokens), two
// to a word
template <int IDT, int ODT, int THREADS, int VECTORS, bool WIDE, bool IN_PLACE>
__global__ __launch_bounds__(THREADS) void adjust_logits_kernel(AdjustParams p) {
  constexpr int kVectors = VECTORS;
  constexpr int kRange = THREADS * kVectors * 8;  // tokens of a work-group
  constexpr int kCountWords = WIDE ? kRange : kRange / 2;
  constexpr uint32_t kInPrompt = WIDE ? 0x80000000u : 0x8000u;
  extern __shared__ __attribute__((aligned(16))) uint32_t counts[];  // [kCountWords], then [kRange] bias entries + 1
  uint32_t* const entries = counts + (p.history ? kCountWords : 0);
  // all arguments in one batch, before anything waits for one of them
  asm volatile("" ::"s"(p.logits), "s"(p.ld), "s"(p.out), "s"(p.ld_out), "s"(p.rows), "s"(p.vocab), "s"(p.history),
               "s"(p.row_seq), "s"(p.bias_start), "s"(p.allowed), "s"(p.allowed_rows));
  const int row = blockIdx.z * kRowsPerSlice + blockIdx.y;
  if (row >= p.rows) return;
  const int base = blockIdx.x * kRange;
  const int tid = threadIdx.x;
  const bool counted = p.history != nullptr, biased = p.bias_start != nullptr;

  // Logits are on their way while the history is counted: all of them, or those that the mask
  // does not ban; in place, only those that change are read at all, later.  The row's last
  // vocab % 8 are taken one by one at the end.
  Raw<IDT> raw[kVectors];
  uint32_t bits[kVectors];  // of this thread's tokens in the mask
  auto token_of = [&](int v) { return base + (v * THREADS + tid) * 8; };
#pragma unroll
  for (int v = 0; v < kVectors; ++v) bits[v] = 0xFFu;
  if (p.allowed) {
    const int mask = p.allowed_rows ? ((ConstI32*)p.allowed_rows)[row] : row;
    if (mask >= 0) {
#pragma unroll
      for (int v = 0; v < kVectors; ++v)
        bits[v] = mask < p.num_allowed && token_of(v) < p.vocab ? p.allowed[mask * p.allowed_stride + token_of(v) / 8] : 0u;
    }
  }
  if constexpr (!IN_PLACE) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (bits[v] && token_of(v) + 8 <= p.vocab) raw[v] = load8<IDT>(p.logits, (int64_t)row * p.ld + token_of(v));
  }

  if (counted || biased) {
    const int words = (counted ? kCountWords : 0) + (biased ? kRange : 0);
    for (int i = tid * 4; i < words; i += THREADS * 4) *(u32x4*)(counts + i) = u32x4{0, 0, 0, 0};
    lds_barrier();
  }
  const uint32_t limit = (uint32_t)min(kRange, p.vocab - base);
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  const int seq = counted && p.row_seq ? ((ConstI32*)p.row_seq)[row] : row;
  if (counted && seq >= 0 && seq < p.num_seqs) {
    repetition = p.repetitions ? ((ConstF32*)p.repetitions)[row] : p.repetition;
    presence = p.presences ? ((ConstF32*)p.presences)[row] : p.presence;
    frequency = p.frequencies ? ((ConstF32*)p.frequencies)[row] : p.frequency;
    const int32_t* tokens = p.history + (int64_t)seq * p.history_stride;
    typedef int32_t vec __attribute__((ext_vector_type(4), aligned(4)));
    vec first;  // of this thread, loaded before the length is known
    const bool ahead = tid * 4 + 4 <= p.capacity;
    if (ahead) first = *(const vec*)(tokens + tid * 4);
    const int len = min(max(((ConstI32*)p.history_len)[seq], 0), p.capacity);
    const int prompt = p.prompt_len ? min(max(((ConstI32*)p.prompt_len)[seq], 0), len) : 0;
    auto seen = [&](int token) {
      const uint32_t u = (uint32_t)(token - base);
      if (u < limit) atomicOr(&counts[WIDE ? u : u / 2], WIDE ? kInPrompt : kInPrompt << u % 2 * 16);
    };
    auto made = [&](int token) {
      const uint32_t u = (uint32_t)(token - base);
      if (u < limit) atomicAdd(&counts[WIDE ? u : u / 2], WIDE ? 1u : 1u << u % 2 * 16);
    };
    const int guesses = p.drafts && p.row_drafts ? min(((ConstI32*)p.row_drafts)[row], p.max_drafts) : 0;
    const int32_t* drafts = p.drafts + (int64_t)seq * p.max_drafts;
    const int guess = tid < guesses ? drafts[tid] : -1;
    // sixteen tokens per thread in flight
    constexpr int kStep = THREADS * 4, kBatch = 4;
    auto count = [&](const vec& t, int at) {
      if (at + 4 <= prompt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) seen(t[e]);
      } else if (at >= prompt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) made(t[e]);
      } else {
        for (int e = 0; e < 4; ++e) at + e < prompt ? seen(tokens[at + e]) : made(tokens[at + e]);
      }
    };
    int i = tid * 4;
    if (ahead && i + 4 <= len) {
      count(first, i);
      i += kStep;
    }
    for (; i + (kBatch - 1) * kStep + 4 <= len; i += kBatch * kStep) {
      vec t[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) t[j] = *(const vec*)(tokens + i + j * kStep);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) count(t[j], i + j * kStep);
    }
    for (; i < len; i += kStep) {
      if (i + 4 <= len) {
        count(*(const vec*)(tokens + i), i);
      } else {
        for (int e = i; e < len; ++e) e < prompt ? seen(tokens[e]) : made(tokens[e]);
      }
    }
    if (tid < guesses) made(guess);
    for (int j = tid + THREADS; j < guesses; j += THREADS) made(drafts[j]);
  }
  if (biased) {  // of a token listed twice the last entry counts
    const int from = max(((ConstI32*)p.bias_start)[row], 0), to = min(((ConstI32*)p.bias_start)[row + 1], p.num_biases);
    for (int i = from + tid; i < to; i += THREADS) {
      const uint32_t u = (uint32_t)(p.bias_tokens[i] - base);
      if (u < limit) atomicMax(&entries[u], (uint32_t)i + 1);
    }
  }
  if (counted || biased) lds_barrier();
  if (!(repetition > 0.f && repetition < __builtin_inff())) repetition = 1.f;
  if (presence != presence) presence = 0.f;
  if (frequency != frequency) frequency = 0.f;

  auto adjusted = [&](float x, uint32_t word, uint32_t entry, uint32_t bit) {
    if (word != 0) {
      x = x > 0.f ? x / repetition : x * repetition;
      const uint32_t n = word & ~kInPrompt;
      if (n != 0) x -= frequency * (float)n + presence;
    }
    if (entry != 0) x += p.bias_values[entry - 1];
    return bit ? x : -__builtin_inff();
  };
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int local = (v * THREADS + tid) * 8;
    const int token = base + local;
    if (token + 8 <= p.vocab) {
      u32x4 c[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}}, b[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
      if (counted) {
        c[0] = *(const u32x4*)(counts + (WIDE ? local : local / 2));
        if (WIDE) c[1] = *(const u32x4*)(counts + local + 4);
      }
      if (biased) {
        b[0] = *(const u32x4*)(entries + local);
        b[1] = *(const u32x4*)(entries + local + 4);
      }
      const u32x4 any = c[0] | c[1] | b[0] | b[1];
      const bool touched = (any[0] | any[1] | any[2] | any[3]) != 0;
      if constexpr (IN_PLACE) {
        if (!touched && bits[v] == 0xFFu) continue;
        if (bits[v]) raw[v] = load8<IDT>(p.logits, (int64_t)row * p.ld + token);
      }
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = value_of(raw[v], e);
      if (touched) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t word = WIDE ? c[e / 4][e % 4] : e % 2 ? c[0][e / 2] >> 16 : c[0][e / 2] & 0xFFFFu;
          x[e] = adjusted(x[e], word, b[e / 4][e % 4], 1);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(bits[v] >> e & 1)) x[e] = -__builtin_inff();
      store8<ODT>(p.out, (int64_t)row * p.ld_out + token, x);
    } else {
      for (int e = 0; token + e < p.vocab; ++e) {
        const float x = load_scale<IDT>(p.logits, (int64_t)row * p.ld + token + e);
        const int at = local + e;
        uint32_t word = 0;
        if (counted) word = WIDE ? counts[at] : counts[at / 2] >> at % 2 * 16 & 0xFFFFu;
        store_scale<ODT>(p.out, (int64_t)row * p.ld_out + token + e,
                         adjusted(x, word, biased ? entries[at] : 0, bits[v] >> e & 1));
      }
    }
  }
}

template <int IDT, int ODT, int THREADS, int VECTORS, bool WIDE>
int launch_ranges(const AdjustParams& p, hipStream_t stream) {
  constexpr int kRange = THREADS * VECTORS * 8;
  NE_CHECK_SUPPORTED(p.rows <= kRowsPerSlice * 65535, "too many rows: %d", p.rows);
  const dim3 grid(ceil_div(p.vocab, kRange), p.rows < kRowsPerSlice ? p.rows : kRowsPerSlice, ceil_div(p.rows, kRowsPerSlice));
  const size_t lds = (p.history ? kRange * (WIDE ? 4 : 2) : 0) + (p.bias_start ? kRange * 4 : 0);
  if constexpr (IDT == ODT) {
    if (p.out == p.logits) {
      hipLaunchKernelGGL((adjust_logits_kernel<IDT, ODT, THREADS, VECTORS, WIDE, true>), grid, dim3(THREADS), lds, stream, p);
      return check_launch("adjust_logits");
    }
  }
  hipLaunchKernelGGL((adjust_logits_kernel<IDT, ODT, THREADS, VECTORS, WIDE, false>), grid, dim3(THREADS), lds, stream, p);
  return check_launch("adjust_logits");
}

// 8,192 tokens per work-group, 4,096 where that leaves CUs idle: one row of 151,936 (20 biases) 5.7 and
// 4.5 us, 320 rows with histories of up to 2,048 tokens 48 and 61.  Histories that need wide counters
// are read by 16 waves, 16 rows of 32,003 with up to 120,000 tokens in 16.6 us (8 waves 21-23).
template <int IDT, int ODT>
int launch_adjust(const AdjustParams& p, hipStream_t stream) {
  if (p.history && (int64_t)p.capacity + p.max_drafts > kMaxNarrow) return launch_ranges<IDT, ODT, 1024, 1, true>(p, stream);
  if ((int64_t)p.rows * ceil_div(p.vocab, 8192) <= 2 * kNumCu) return launch_ranges<IDT, ODT, 512, 1, false>(p, stream);
  return launch_ranges<IDT, ODT, 512, 2, false>(p, stream);
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
