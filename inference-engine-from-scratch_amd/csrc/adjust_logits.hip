// Logits under penalties for repeated tokens, biases of single tokens and masks of allowed ones,
// before sampling or acceptance.  Per row, with c the token's occurrences in the row's output (the
// history after the prompt, and the guesses before the row in a verify step) and "seen" anywhere:
//   x1 = seen ? (x > 0 ? x / r : x r) : x     repetition
//   x2 = x1 - (f c + p [c > 0])               frequency and presence
//   x3 = x2 + bias,  x4 = allowed ? x3 : -inf
// in fp32, rounded once to the output's type.
//
// The counts need no state from step to step: they come from the history itself, which the
// caller holds anyway.  A work-group owns a range of one row's tokens (4,096 or 8,192), counts the
// history's tokens of its range in LDS (integer atomics: their order does not matter) while its
// logits are on their way to registers, and applies everything in one pass over them.  So a history
// is read once per range (19 or 38 times for 151,936 tokens), after the first from the L2s.
//
// A token has 16 bits of a table of counts: the output count below, "in the prompt" in the top bit;
// and 16 bits of a second table for its bias, the entry's number in the row's list, so that of two
// entries for one token the later one wins whatever the order of the lanes.  Histories of more than
// 32,767 tokens and lists of more than 65,534 biases take words instead.  Half the LDS leaves room
// for more work-groups per CU: 64 rows of 151,936 with 8 biases each and histories of up to 4,096 tokens,
// bf16 to fp32, took 16.9 us with 16 bits for both against 18.3 with words for the biases.
//
// Tokens of other ranges count into a spare word of their lane, which takes three instructions where
// leaving their lanes out takes five; a wave knows from its first token which side of the prompt's end it
// is on, and has four loads in flight.  That is 16.0 us for those 64 rows, and 44.0 against 48 for 320
// rows in bf16 behind histories of up to 2,048 tokens.
//
// Bound by memory where rows are many: the 64 rows move 58 MB (3.6 TB/s), the 320 rows 195 MB (4.4
// TB/s; a copy of 1 GiB reaches 5.1).  One row (4.5 us) is the latency of its chain: arguments, history
// length, history, counts, stores.  Long histories of repetitive text are bound by LDS atomics on
// the same tokens: 16 rows of 32,003 with up to 120,000 tokens, the commonest of them 7.5 %, take 16.4 us
// (12.9 where all tokens are alike and in the caches, 5.7 without a history; the logits alone 1.7).
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
constexpr int kMaxNarrowCount = 32767, kMaxNarrowBias = 65534;
constexpr int kRowsPerSlice = 32767;  // of the grid

// VEC values as they lie in memory, from any element's address (global accesses need not be
// aligned): 16 bytes of the wider of the two types, so that a wave's loads and stores are both
// contiguous.
template <int DT, int VEC>
struct Raw {
  static constexpr int kWords = DT == NE_DTYPE_FP32 ? VEC : VEC / 2;
  typedef uint32_t vec __attribute__((ext_vector_type(kWords), aligned(2)));
  vec word;
};

template <int DT>
__device__ __forceinline__ const void* element(const void* p, int64_t i) {
  return (const char*)p + i * (DT == NE_DTYPE_FP32 ? 4 : 2);
}

template <int DT, int VEC>
__device__ __forceinline__ float value_of(const Raw<DT, VEC>& r, int e) {
  if constexpr (DT == NE_DTYPE_FP32) {
    return __uint_as_float(r.word[e]);
  } else {
    const uint32_t half = e % 2 ? r.word[e / 2] >> 16 : r.word[e / 2] & 0xFFFFu;
    return DT == NE_DTYPE_BF16 ? bf16_to_f32((uint16_t)half) : f16_to_f32((uint16_t)half);
  }
}

template <int DT, int VEC>
__device__ __forceinline__ void store_values(void* p, int64_t i, const float (&f)[VEC]) {
  Raw<DT, VEC> r;
#pragma unroll
  for (int w = 0; w < Raw<DT, VEC>::kWords; ++w) {
    if constexpr (DT == NE_DTYPE_FP32) {
      r.word[w] = __float_as_uint(f[w]);
    } else if constexpr (DT == NE_DTYPE_BF16) {
      r.word[w] = pack_bf16x2(f[2 * w], f[2 * w + 1]);
    } else {
      r.word[w] = (uint32_t)f32_to_f16(f[2 * w]) | (uint32_t)f32_to_f16(f[2 * w + 1]) << 16;
    }
  }
  *(typename Raw<DT, VEC>::vec*)element<DT>(p, i) = r.word;
}

// A token's entry in an LDS table: a word, or (narrow) half of one.
template <bool WIDE>
__device__ __forceinline__ uint32_t entry_of(const uint32_t* table, int i) {
  return WIDE ? table[i] : table[i / 2] >> i % 2 * 16 & 0xFFFFu;
}

// VEC entries from a multiple of VEC on
template <bool WIDE, int VEC>
struct Entries {
  uint32_t word[WIDE ? VEC : VEC / 2];
  __device__ __forceinline__ void read(const uint32_t* table, int i) {
    constexpr int kWords = WIDE ? VEC : VEC / 2;
    typedef uint32_t vec __attribute__((ext_vector_type(kWords > 4 ? 4 : kWords)));
#pragma unroll
    for (int w = 0; w < kWords; w += 4) {
      const vec v = *(const vec*)(table + (WIDE ? i : i / 2) + w);
#pragma unroll
      for (int e = 0; e < 4 && w + e < kWords; ++e) word[w + e] = v[e];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t& w : word) w = 0;
  }
  __device__ __forceinline__ uint32_t any() const {
    uint32_t a = 0;
#pragma unroll
    for (uint32_t w : word) a |= w;
    return a;
  }
  __device__ __forceinline__ uint32_t at(int e) const {
    return WIDE ? word[WIDE ? e : 0] : e % 2 ? word[e / 2] >> 16 : word[e / 2] & 0xFFFFu;
  }
};

struct Penalties {
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  __device__ __forceinline__ void read(const AdjustParams& p, int row) {
    repetition = p.repetitions ? ((ConstF32*)p.repetitions)[row] : p.repetition;
    presence = p.presences ? ((ConstF32*)p.presences)[row] : p.presence;
    frequency = p.frequencies ? ((ConstF32*)p.frequencies)[row] : p.frequency;
  }
  __device__ __forceinline__ void check() {
    if (!(repetition > 0.f && repetition < __builtin_inff())) repetition = 1.f;
    if (presence != presence) presence = 0.f;
    if (frequency != frequency) frequency = 0.f;
  }
  // of a token that was seen, n times in the output
  __device__ __forceinline__ float apply(float x, uint32_t n) const {
    x = x > 0.f ? x / repetition : x * repetition;
    if (n != 0) x -= frequency * (float)n + presence;
    return x;
  }
};

// WIDE: tables of 32-bit words; otherwise of 16 bits (histories of at most kMaxNarrowCount tokens and
// at most kMaxNarrowBias biases).
template <int IDT, int ODT, int THREADS, int VECTORS, bool WIDE, bool IN_PLACE>
__global__ __launch_bounds__(THREADS) void adjust_logits_kernel(AdjustParams p) {
  constexpr int VEC = ODT == NE_DTYPE_FP32 ? 4 : 8;
  constexpr int kVectors = VECTORS * 8 / VEC;
  constexpr int kRange = THREADS * VECTORS * 8;  // tokens of a work-group
  constexpr int kTableWords = WIDE ? kRange : kRange / 2;
  constexpr int kCountWords = kTableWords + kWave;  // and a spare word per lane, for tokens of other ranges
  constexpr uint32_t kInPrompt = WIDE ? 0x80000000u : 0x8000u;
  extern __shared__ __attribute__((aligned(16))) uint32_t counts[];  // [kCountWords], then the bias entries' numbers [kTableWords]
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
  // vocab % VEC are taken one by one at the end.
  Raw<IDT, VEC> raw[kVectors];
  uint32_t bits[kVectors];  // of this thread's tokens in the mask
  auto token_of = [&](int v) { return base + (v * THREADS + tid) * VEC; };
#pragma unroll
  for (int v = 0; v < kVectors; ++v) bits[v] = (1u << VEC) - 1;
  if (p.allowed) {
    const int mask = p.allowed_rows ? ((ConstI32*)p.allowed_rows)[row] : row;
    if (mask >= 0) {
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        bits[v] = mask < p.num_allowed && token_of(v) < p.vocab ? p.allowed[mask * p.allowed_stride + token_of(v) / 8] : 0u;
        if (VEC == 4) bits[v] = bits[v] >> token_of(v) % 8 & 0xFu;
      }
    }
  }
  auto load = [&](int v) {
    raw[v].word = *(const typename Raw<IDT, VEC>::vec*)element<IDT>(p.logits, (int64_t)row * p.ld + token_of(v));
  };
  if constexpr (!IN_PLACE) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (bits[v] && token_of(v) + VEC <= p.vocab) load(v);
  }

  if (counted || biased) {
    const int words = (counted ? kCountWords : 0) + (biased ? kTableWords : 0);
    for (int i = tid * 4; i < words; i += THREADS * 4) *(u32x4*)(counts + i) = u32x4{0, 0, 0, 0};
    lds_barrier();
  }
  const uint32_t limit = (uint32_t)min(kRange, p.vocab - base);
  Penalties penalties;
  const int seq = counted && p.row_seq ? ((ConstI32*)p.row_seq)[row] : row;
  if (counted && seq >= 0 && seq < p.num_seqs) {
    penalties.read(p, row);
    const int32_t* tokens = p.history + (int64_t)seq * p.history_stride;
    typedef int32_t vec __attribute__((ext_vector_type(4), aligned(4)));
    vec first;  // of this thread, loaded before the length is known
    const bool ahead = tid * 4 + 4 <= p.capacity;
    if (ahead) first = *(const vec*)(tokens + tid * 4);
    const int len = min(max(((ConstI32*)p.history_len)[seq], 0), p.capacity);
    const int prompt = p.prompt_len ? min(max(((ConstI32*)p.prompt_len)[seq], 0), len) : 0;
    const int lane = tid % kWave;
    const uint32_t spare = kRange + (WIDE ? lane : 2 * lane);
    auto seen = [&](int token) {
      const uint32_t u = min((uint32_t)(token - base), spare);
      atomicOr(&counts[WIDE ? u : u / 2], WIDE ? kInPrompt : kInPrompt << u % 2 * 16);
    };
    auto made = [&](int token) {
      const uint32_t u = min((uint32_t)(token - base), spare);
      atomicAdd(&counts[WIDE ? u : u / 2], WIDE ? 1u : 1u << u % 2 * 16);
    };
    const int guesses = p.drafts && p.row_drafts ? min(((ConstI32*)p.row_drafts)[row], p.max_drafts) : 0;
    const int32_t* drafts = p.drafts + (int64_t)seq * p.max_drafts;
    const int guess = tid < guesses ? drafts[tid] : -1;
    const int whole = len & ~3;  // in vectors; the last len % 4 by a thread each
    const int last = tid < len - whole ? tokens[whole + tid] : -1;
    // A wave takes 256 consecutive tokens at a time, kBatch such loads in flight; lanes past the
    // end count the token -1, which no range has.
    constexpr int kStep = THREADS * 4, kBatch = 4;
    auto count = [&](const vec& t, int w) {
      if (w + kWave * 4 <= prompt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) seen(t[e]);
      } else if (w >= prompt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) made(t[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) w + lane * 4 + e < prompt ? seen(t[e]) : made(t[e]);
      }
    };
    auto cut = [&](vec& t, int w) {
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = w + lane * 4 < whole ? t[e] : -1;
    };
    int w = __builtin_amdgcn_readfirstlane(tid / kWave) * (kWave * 4);
    if (w < whole) {
      cut(first, w);
      count(first, w);
      w += kStep;
    }
    vec t[kBatch];
    for (; w + (kBatch - 1) * kStep + kWave * 4 <= whole; w += kBatch * kStep) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) t[j] = *(const vec*)(tokens + w + j * kStep + lane * 4);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) count(t[j], w + j * kStep);
    }
    if (w < whole) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) t[j] = *(const vec*)(tokens + min(w + j * kStep + lane * 4, whole - 4));
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (w + j * kStep < whole) {
          cut(t[j], w + j * kStep);
          count(t[j], w + j * kStep);
        }
    }
    if (tid < len - whole) whole + tid < prompt ? seen(last) : made(last);
    if (tid < guesses) made(guess);
    for (int j = tid + THREADS; j < guesses; j += THREADS) made(drafts[j]);
  }
  int from = 0;  // of the row's biases; of a token listed twice the last entry counts
  if (biased) {
    from = max(((ConstI32*)p.bias_start)[row], 0);
    const int to = min(((ConstI32*)p.bias_start)[row + 1], p.num_biases);
    for (int i = from + tid; i < to; i += THREADS) {
      const uint32_t u = (uint32_t)(p.bias_tokens[i] - base);
      if (u >= limit) continue;
      if constexpr (WIDE) {
        atomicMax(&entries[u], (uint32_t)(i - from) + 1);
      } else {  // the larger number into half of a word
        uint32_t* const word = &entries[u / 2];
        const int shift = u % 2 * 16;
        uint32_t old = *word;
        while ((old >> shift & 0xFFFFu) < (uint32_t)(i - from) + 1) {
          const uint32_t is = atomicCAS(word, old, (old & ~(0xFFFFu << shift)) | (uint32_t)(i - from + 1) << shift);
          if (is == old) break;
          old = is;
        }
      }
    }
  }
  if (counted || biased) lds_barrier();
  penalties.check();

  auto adjusted = [&](float x, uint32_t word, uint32_t entry, uint32_t bit) {
    if (word != 0) x = penalties.apply(x, word & ~kInPrompt);
    if (entry != 0) x += p.bias_values[from + (int)entry - 1];
    return bit ? x : -__builtin_inff();
  };
#pragma unroll
  for (int v = 0; v < kVectors; ++v) {
    const int local = (v * THREADS + tid) * VEC;
    const int token = base + local;
    if (token + VEC <= p.vocab) {
      Entries<WIDE, VEC> c, b;
      c.clear();
      b.clear();
      if (counted) c.read(counts, local);
      if (biased) b.read(entries, local);
      const bool touched = (c.any() | b.any()) != 0;
      if constexpr (IN_PLACE) {
        if (!touched && bits[v] == (1u << VEC) - 1) continue;
        if (bits[v]) load(v);
      }
      float x[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = value_of(raw[v], e);
      if (touched) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = adjusted(x[e], c.at(e), b.at(e), 1);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (!(bits[v] >> e & 1)) x[e] = -__builtin_inff();
      store_values<ODT, VEC>(p.out, (int64_t)row * p.ld_out + token, x);
    } else {
      for (int e = 0; token + e < p.vocab; ++e) {
        const float x = load_scale<IDT>(p.logits, (int64_t)row * p.ld + token + e);
        store_scale<ODT>(p.out, (int64_t)row * p.ld_out + token + e,
                         adjusted(x, counted ? entry_of<WIDE>(counts, local + e) : 0,
                                  biased ? entry_of<WIDE>(entries, local + e) : 0, bits[v] >> e & 1));
      }
    }
  }
}

template <int IDT, int ODT, int THREADS, int VECTORS, bool WIDE, bool IN_PLACE>
int launch_kernel(const AdjustParams& p, hipStream_t stream) {
  constexpr int kRange = THREADS * VECTORS * 8, kTable = kRange * (WIDE ? 4 : 2), kSpare = kWave * 4;
  NE_CHECK_SUPPORTED(p.rows <= kRowsPerSlice * 65535, "too many rows: %d", p.rows);
  const auto kernel = adjust_logits_kernel<IDT, ODT, THREADS, VECTORS, WIDE, IN_PLACE>;
  if constexpr (2 * kTable + kSpare > 64 * 1024) {  // more than the default dynamic LDS, once per instantiation
    static const hipError_t attr = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * kTable + kSpare);
    if (attr != hipSuccess) {
      set_error("adjust_logits: cannot reserve %d bytes of LDS: %s", 2 * kTable + kSpare, hipGetErrorString(attr));
      return NE_ELAUNCH;
    }
  }
  const dim3 grid(ceil_div(p.vocab, kRange), p.rows < kRowsPerSlice ? p.rows : kRowsPerSlice, ceil_div(p.rows, kRowsPerSlice));
  const size_t lds = (p.history ? kTable + kSpare : 0) + (p.bias_start ? kTable : 0);
  hipLaunchKernelGGL(kernel, grid, dim3(THREADS), lds, stream, p);
  return check_launch("adjust_logits");
}

template <int IDT, int ODT, int THREADS, int VECTORS, bool WIDE>
int launch_ranges(const AdjustParams& p, hipStream_t stream) {
  if constexpr (IDT == ODT) {
    if (p.out == p.logits) return launch_kernel<IDT, ODT, THREADS, VECTORS, WIDE, true>(p, stream);
  }
  return launch_kernel<IDT, ODT, THREADS, VECTORS, WIDE, false>(p, stream);
}

// Penalties alone, in place: only tokens of the history change, and a work-group takes a row's in one
// pass: 320 rows with 2,000 tokens each read 19.6 and write 14.8 MB (6.8 us at a copy's rate) in 19.7-21.5; the rest
// is its chain, length, history, table and scattered logits.  An LDS table of 2^size slots, at least 1.5 times the tokens, takes each of them by linear probing
// (so a free slot ends every search), its counts beside it; then each slot's logit is adjusted.
constexpr int kSeenThreads = 512, kMaxSeen = 5461;  // tokens in a table of 8,192 slots, 64 KiB
template <int DT>
__global__ __launch_bounds__(kSeenThreads) void adjust_seen_kernel(AdjustParams p, int size) {
  extern __shared__ __attribute__((aligned(16))) uint32_t tokens_of[];  // [slots] token + 1, 0: free; then the counts
  const int slots = 1 << size;
  uint32_t* const counts = tokens_of + slots;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int seq = p.row_seq ? ((ConstI32*)p.row_seq)[row] : row;
  if (seq < 0 || seq >= p.num_seqs) return;
  const int32_t* const tokens = p.history + (int64_t)seq * p.history_stride;
  typedef int32_t vec __attribute__((ext_vector_type(4), aligned(4)));
  vec first;  // of this thread, loaded before the length is known
  if (tid * 4 + 4 <= p.capacity) first = *(const vec*)(tokens + tid * 4);
  for (int i = tid * 4; i < 2 * slots; i += kSeenThreads * 4) *(u32x4*)(tokens_of + i) = u32x4{0, 0, 0, 0};
  const int len = min(max(((ConstI32*)p.history_len)[seq], 0), p.capacity);
  const int prompt = p.prompt_len ? min(max(((ConstI32*)p.prompt_len)[seq], 0), len) : 0;
  const int guesses = p.drafts && p.row_drafts ? min(((ConstI32*)p.row_drafts)[row], p.max_drafts) : 0;
  Penalties penalties;
  penalties.read(p, row);
  lds_barrier();
  auto add = [&](int token, bool in_prompt) {
    if ((uint32_t)token >= (uint32_t)p.vocab) return;
    const uint32_t key = (uint32_t)token + 1;
    uint32_t at = (uint32_t)token * 2654435761u >> (32 - size);
    for (;;) {
      uint32_t is = *(volatile uint32_t*)&tokens_of[at];  // repeated tokens read it side by side
      if (is == 0) is = atomicCAS(&tokens_of[at], 0u, key);
      if (is == 0 || is == key) break;
      at = (at + 1) & (slots - 1);
    }
    if (in_prompt) {
      atomicOr(&counts[at], 0x80000000u);
    } else {
      atomicAdd(&counts[at], 1u);
    }
  };
  for (int i = tid * 4; i < len; i += kSeenThreads * 4) {
    if (i + 4 <= len) {
      const vec t = i == tid * 4 ? first : *(const vec*)(tokens + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) add(t[e], i + e < prompt);
    } else {
      for (int e = i; e < len; ++e) add(tokens[e], e < prompt);
    }
  }
  const int32_t* const drafts = p.drafts + (int64_t)seq * p.max_drafts;
  for (int i = tid; i < guesses; i += kSeenThreads) add(drafts[i], false);
  lds_barrier();
  penalties.check();
  constexpr int kBatch = 4;
  for (int i = tid; i < slots; i += kSeenThreads * kBatch) {
    uint32_t key[kBatch];
    float x[kBatch];
    int64_t at[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int slot = i + j * kSeenThreads;
      key[j] = slot < slots ? tokens_of[slot] : 0;
      at[j] = (int64_t)row * p.ld + key[j] - 1;
      if (key[j]) x[j] = load_scale<DT>(p.logits, at[j]);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (key[j]) store_scale<DT>(p.out, at[j], penalties.apply(x[j], counts[i + j * kSeenThreads] & 0x7FFFFFFFu));
  }
}

template <int DT>
int launch_seen(const AdjustParams& p, hipStream_t stream) {
  int size = 9;
  while ((2 << size) < 3 * (p.capacity + p.max_drafts)) ++size;
  const size_t lds = (size_t)8 << size;
  hipLaunchKernelGGL(adjust_seen_kernel<DT>, dim3(p.rows), dim3(kSeenThreads), lds, stream, p, size);
  return check_launch("adjust_logits");
}

// In place under penalties alone a row's own tokens are cheaper than its vocabulary where rows are many and
// histories short beside it (us, bf16, ranges / own tokens): 320 rows of 151,936, histories of their own in buffers of
// 2,048 tokens, with 100 tokens 23.6 / 6.5, with 2,000 36.6 / 21.5, 64 rows with 2,000 of 4,096 11.3 / 10.5; but 320 rows
// with 8,000 of 8,192 50 / 83, one row with 600 4.9 / 6.3, 320 rows of 9,001 with 2,000 9.8 / 10.7.
//
// The host knows a buffer's width, not the lengths in it, so every rule here goes by the width, and what a
// short history costs depends on it: 64 sequences' 320 verify rows with 100 tokens take 5.6 us in a buffer of 108, 8.3
// in one of 4,101 and 38.7 in one of 40,965 (32-bit tables), with 2,000 tokens 19.7 (of 2,008), 20.3 and 49.3.
//
// 8,192 tokens per work-group, 4,096 where that leaves CUs idle: one row of 151,936 (20 biases) 5.7 and
// 4.5 us, 320 rows with histories of up to 2,048 tokens 44 and 53.  Histories that need wide counters
// are read by 16 waves, 16 rows of 32,003 with up to 120,000 tokens in 16.4 us (8 waves 17.6 and 19.6).
template <int IDT, int ODT>
int launch_adjust(const AdjustParams& p, hipStream_t stream) {
  if constexpr (IDT == ODT) {
    const int64_t tokens = (int64_t)p.capacity + p.max_drafts;
    if (p.out == p.logits && p.history && !p.bias_start && !p.allowed && tokens <= kMaxSeen && p.vocab > 16 * tokens &&
        (int64_t)p.rows * ceil_div(p.vocab, 8192) > 2 * kNumCu && p.rows < (1 << 22))
      return launch_seen<IDT>(p, stream);
  }
  const bool wide = p.history && (int64_t)p.capacity + p.max_drafts > kMaxNarrowCount;
  if (wide || (p.bias_start && p.num_biases > kMaxNarrowBias)) return launch_ranges<IDT, ODT, 1024, 1, true>(p, stream);
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
