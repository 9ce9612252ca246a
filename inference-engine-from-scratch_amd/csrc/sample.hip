// Sampling a token per row of logits from a given uniform, under temperature, top-k,
// top-p and min-p, and the filtered distribution itself.
//
// Definition.  A row's tokens are ordered by logit (descending), then by index
// (ascending); NaN and -inf are no tokens.  y = x log2(e) / T; a token's weight is
// 2^(y - Y) with one Y per row.  Kept: the first n = min(n_k, n_p, n_m) tokens of the order,
//   n_k = top_k (all, where top_k is 0 or less),
//   n_p = the fewest whose weight reaches top_p times the weight of the first n_k
//         (all, where top_p is 1 or more),
//   n_m = the tokens with weight at least min_p times the largest,
// and at least one.  The token drawn is the first whose running weight exceeds
// u * (kept weight).  T = 0 keeps the first token alone.
//
// Weights are integers, rint(2^(y - Y) * 2^S) with 2^S * vocab <= 2^63, computed in 64-bit
// floating point: a sum of them does not depend on its order (so neither on the work split
// nor on atomics), and a border between two tokens is off by at most ~2^-S of the row's
// largest weight per token (S = 45 for 151,936 tokens).  32-bit weights would move every
// border of a flat row by 1e-7, a wrong token in a hundred rows of 100,000 tokens.
//
// Three kernels.
//   scan   rows x chunks: reads the logits once.  Per 1 KB segment the largest key; per
//          chunk the first largest token and a histogram over y in steps of 1/16 (1,024
//          bins below the chunk's own base Y, counts and, unless top-k is short, weights).
//          The base is an integer, so histograms of unlike bases merge by shifting 16 bins
//          and one bit per step.
//   pick   one work-group per row: merges the row's histograms, finds the last bin that can
//          hold a kept token, and, where at most 4,096 tokens lie above its end, gathers
//          them (only from segments whose largest key reaches it), sorts them in LDS and
//          finishes there.  A wide nucleus is handled bin by bin: the border of each filter
//          and the draw lie in one bin each, whose tokens are gathered and sorted; a bin
//          with more tokens than the list holds is narrowed by key first, and a run of
//          equal logits by index.
//   probs  rows x chunks: kept weight / sum per token, if asked for.
// What bounds it: one read of the logits (scan), its ~25 64-bit operations per element
// (full rate on this chip), and the chain of round trips in pick.
#include <math.h>
#include <string.h>

#include "ne_common.hpp"

namespace ne {

namespace {

// A token's bin and remainder come from one rounded product in every kernel: no contraction.
#pragma clang fp contract(off)

typedef unsigned long long u64;

constexpr int kBins = 1024;
constexpr int kBinsPerLog2 = 16;
constexpr int kScanThreads = 512;
constexpr int kScanWaves = kScanThreads / kWave;
constexpr int kScanSegs = 2;          // segments per wave and iteration
constexpr int kPickThreads = 512;
constexpr int kPickWaves = kPickThreads / kWave;
constexpr int kList = 4096;           // tokens that pick sorts in LDS
constexpr int kShortTopK = 1024;      // up to here the scan counts tokens and leaves their weights to pick
constexpr int kSub = 2048;            // buckets of a narrowing pass
constexpr int kMaxVocab = 1 << 20;
constexpr int kRowBatch = 1024;       // rows per launch: bounds the workspace

// One chunk's result; its histogram follows in arrays of their own.
struct ChunkHead {
  u64 best;     // first largest token (key, ~index); 0: no token
  double base;  // Y
  uint32_t tokens;
  uint32_t pad[3];
};
// One row's result, for the probs kernel.
struct RowResult {
  u64 last;    // order word of the last kept token; 0: none
  double base;
  double sum;  // kept weight
  double scale;  // 16 log2(e) / T; negative: greedy
};

struct SampleParams {
  const void* logits;
  int64_t ld;
  int32_t rows, vocab;
  int32_t chunks, segs;      // per row
  const float* uniforms;
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  float temperature, top_p, min_p;
  int32_t top_k;
  int32_t weight_exp;        // S
  int32_t* tokens;
  float* probs;
  int64_t ld_probs;
  ChunkHead* heads;          // [rows][chunks]
  uint32_t* counts;          // [rows][chunks][kBins]
  u64* weights;              // [rows][chunks][kBins]
  uint32_t* seg_max;         // [rows][segs]
  RowResult* results;        // [rows]
};

// ---- elements ----
template <int DT>
constexpr int kVec = DT == NE_DTYPE_FP32 ? 4 : 8;  // elements per 16 bytes

// Order key of a logit: larger logit, larger key; -0 as +0; 0 for NaN and -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}
// The value that enters the arithmetic: +inf as the largest finite number (tokens at it share the row).
__device__ __forceinline__ double finite(float x) { return (double)fminf(x, 3.402823466e38f); }

__device__ __forceinline__ u64 order_word(uint32_t key, uint32_t index) { return ((u64)key << 32) | (uint32_t)~index; }
__device__ __forceinline__ uint32_t word_index(u64 w) { return ~(uint32_t)w; }
__device__ __forceinline__ uint32_t word_key(u64 w) { return (uint32_t)(w >> 32); }

// A row's elements in 16-byte vectors that start on the 16-byte grid at or before the row;
// element e of vector v is token v * kVec + e - skew.
template <int DT>
struct Row {
  const char* base;  // of the row, any alignment of an element
  int skew, vocab, vecs;
  __device__ Row(const SampleParams& p, int row) {
    constexpr int kEsz = 16 / kVec<DT>;
    base = (const char*)p.logits + (int64_t)row * p.ld * kEsz;
    skew = (int)((uintptr_t)base & 15) / kEsz;
    vocab = p.vocab;
    vecs = (vocab + skew + kVec<DT> - 1) / kVec<DT>;
  }
  // Keys of vector v; 0 for what lies outside the row.
  __device__ __forceinline__ u32x4 raw(int v, bool& whole) const {
    constexpr int kEsz = 16 / kVec<DT>;
    const int t0 = v * kVec<DT> - skew;
    whole = t0 >= 0 && t0 + kVec<DT> <= vocab;
    // an address that is read whatever the vector: its own, or the row's first whole vector's
    u32x4 x = {0, 0, 0, 0};
    if (whole) x = *(const u32x4*)(base + (int64_t)t0 * kEsz);
    return x;
  }
  __device__ __forceinline__ float single(int t) const {
    if (DT == NE_DTYPE_FP32) return ((const float*)base)[t];
    if (DT == NE_DTYPE_FP16) return f16_to_f32(((const uint16_t*)base)[t]);
    return bf16_to_f32(((const uint16_t*)base)[t]);
  }
  // The vector's values, NaN outside the row.
  __device__ __forceinline__ void values(int v, u32x4 x, bool whole, float (&out)[kVec<DT>]) const {
    if (whole) {
#pragma unroll
      for (int e = 0; e < kVec<DT>; ++e) {
        if constexpr (DT == NE_DTYPE_FP32) {
          const uint32_t bits = x[e];  // (a bit cast of the vector's element itself reads element 0)
          out[e] = __builtin_bit_cast(float, bits);
        } else {
          const uint16_t h = (uint16_t)(x[e / 2] >> (16 * (e & 1)));
          out[e] = DT == NE_DTYPE_FP16 ? f16_to_f32(h) : bf16_to_f32(h);
        }
      }
    } else {
      const int t0 = v * kVec<DT> - skew;
#pragma unroll
      for (int e = 0; e < kVec<DT>; ++e) out[e] = t0 + e >= 0 && t0 + e < vocab ? single(t0 + e) : NAN;
    }
  }
};

// ---- row parameters ----
struct RowParams {
  double scale;  // 16 log2(e) / T
  double log2_min_p;  // -inf: off
  float top_p;
  int top_k;     // 0: off
  bool greedy;
  bool weigh;    // the scan sums weights
};
__device__ __forceinline__ RowParams row_params(const SampleParams& p, int row) {
  RowParams r;
  const float t = p.temperatures ? p.temperatures[row] : p.temperature;
  const int k = p.top_ks ? p.top_ks[row] : p.top_k;
  const float m = p.min_ps ? p.min_ps[row] : p.min_p;
  r.top_p = p.top_ps ? p.top_ps[row] : p.top_p;
  r.greedy = !(t > 0.f);
  r.scale = r.greedy ? 0.0 : kBinsPerLog2 * 1.4426950408889634 / (double)t;
  r.top_k = k > 0 && k < p.vocab ? k : 0;
  r.weigh = !r.greedy && (r.top_k == 0 || r.top_k > kShortTopK);
  r.log2_min_p = m > 0.f ? log2(fmin((double)m, 1.0)) : -INFINITY;
  return r;
}

// ---- weights ----
// 2^(j / 16), j = 0..15.  y in sixteenths is split into its floor f (a bin) and r in [0, 1):
// 2^(y - Y) = 2^((f - 16 Y) / 16) * 2^(r / 16); floor and remainder are exact, so a
// token's bin is the same under every base.
__constant__ const double kRoots[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.241857812073484,
    1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993, 1.5422108254079408,
    1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// The token's bin below base (0 = largest y) and its remainder; base > y, up to the rounding of
// values past 2^53 (a temperature next to 0), which the lower bound catches.
__device__ __forceinline__ int bin_of(double y16, double base, double& rem) {
  const double f = floor(y16);
  rem = y16 - f;
  // past kBins - 1: too small to weigh
  return (int)fmin(fmax(kBinsPerLog2 * base - f, 1.0), (double)(1 << 20)) - 1;
}
// 2^(y - Y) for a token of bin b and remainder rem.  2^(rem / 16) by its series around 1 / 32:
// |ln 2 (rem / 16 - 1 / 32)| < 0.0217, whose seventh power over 7! is 4.5e-16.
__device__ __forceinline__ double weight_of(int b, double rem, const double* roots) {
  const int q = b + 1;
  const double z = (rem - 0.5) * (0.6931471805599453 / kBinsPerLog2);
  double e = 1.0 / 720;
  e = fma(e, z, 1.0 / 120);
  e = fma(e, z, 1.0 / 24);
  e = fma(e, z, 1.0 / 6);
  e = fma(e, z, 0.5);
  e = fma(e, z, 1.0);
  e = fma(e, z, 1.0);
  return ldexp(e * (1.0218971486541166 /* 2^(1/32) */ * roots[-q & 15]), -((q + 15) >> 4));
}
// rint(w * 2^S) below 2^52, S <= 51: adding 2^52 leaves the integer in the low mantissa bits
__device__ __forceinline__ u64 weight_int(double w, int s) {
  return __builtin_bit_cast(u64, ldexp(w, s) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ u64 weight_of_key(uint32_t key, const RowParams& r, double base, int s, const double* roots) {
  double rem;
  const int b = bin_of(finite(logit_of(key)) * r.scale, base, rem);
  return b < kBins ? weight_int(weight_of(b, rem, roots), s) : 0;
}

__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 x = __shfl_xor(v, o);
    v = x > v ? x : v;
  }
  return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// ---- scan ----
template <int DT>
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(SampleParams p) {
  constexpr int E = kVec<DT>;
  __shared__ uint32_t s_count[kBins];
  __shared__ u64 s_weight[kBins];
  __shared__ double s_roots[16];
  __shared__ uint32_t s_max[2][kScanWaves];
  __shared__ u64 s_best[kScanWaves];
  __shared__ uint32_t s_tokens;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int row = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x % p.chunks;
  const RowParams r = row_params(p, row);
  const Row<DT> x(p, row);
  const int segs = (x.vecs + kWave - 1) / kWave;
  const int seg0 = (int)((int64_t)segs * chunk / p.chunks);
  const int seg1 = (int)((int64_t)segs * (chunk + 1) / p.chunks);
  if (tid < 16) s_roots[tid] = kRoots[tid];
  if (tid == 0) s_tokens = 0;
#pragma unroll
  for (int b = 0; b < kBins / kScanThreads; ++b) {
    s_count[tid + b * kScanThreads] = 0;
    s_weight[tid + b * kScanThreads] = 0;
  }
  uint32_t best_key = 0, best_index = 0, tokens = 0;
  double base = 0;
  bool any = false;  // base is set
  constexpr int kStep = kScanWaves * kScanSegs;
  u32x4 raw[kScanSegs];
  bool whole[kScanSegs];
  auto load = [&](int s0) {
#pragma unroll
    for (int j = 0; j < kScanSegs; ++j) {
      const int seg = s0 + wave * kScanSegs + j;
      whole[j] = false;
      if (seg < seg1) raw[j] = x.raw(seg * kWave + lane, whole[j]);
    }
  };
  load(seg0);
  int turn = 0;
  for (int s0 = seg0; s0 < seg1; s0 += kStep, turn ^= 1) {
    float val[kScanSegs][E];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kScanSegs; ++j) {
      const int seg = s0 + wave * kScanSegs + j;
      const int v = seg * kWave + lane;
#pragma unroll
      for (int e = 0; e < E; ++e) val[j][e] = NAN;
      uint32_t here = 0;
      if (seg < seg1) {
        if (v < x.vecs) x.values(v, raw[j], whole[j], val[j]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t k = key_of(val[j][e]);
          if (k > best_key) {  // a lane's tokens come in order of index
            best_key = k;
            best_index = v * E + e - x.skew;
          }
          here = max(here, k);
        }
        here = wave_max_u32(here);
        if (lane == 0) p.seg_max[(int64_t)row * p.segs + seg] = here;
      }
      most = max(most, here);
    }
    if (s0 + kStep < seg1) load(s0 + kStep);
    if (lane == 0) s_max[turn][wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) most = max(most, s_max[turn][w]);
    if (r.greedy || most == 0) continue;
    const double top = floor(finite(logit_of(most)) * r.scale / kBinsPerLog2) + 1.0;
    if (!any) {
      base = top;
      any = true;
    } else if (top > base) {  // a larger logit than so far: the bins move down
      const int up = (int)fmin(top - base, (double)(kBins / kBinsPerLog2));
      uint32_t c[kBins / kScanThreads];
      u64 w[kBins / kScanThreads];
#pragma unroll
      for (int b = 0; b < kBins / kScanThreads; ++b) {
        const int from = tid + b * kScanThreads - kBinsPerLog2 * up;
        c[b] = from >= 0 ? s_count[from] : 0;
        w[b] = from >= 0 ? s_weight[from] >> up : 0;
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < kBins / kScanThreads; ++b) {
        s_count[tid + b * kScanThreads] = c[b];
        s_weight[tid + b * kScanThreads] = w[b];
      }
      __syncthreads();
      base = top;
    }
#pragma unroll
    for (int j = 0; j < kScanSegs; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (key_of(val[j][e]) == 0) continue;
        ++tokens;
        double rem;
        const int b = bin_of(finite(val[j][e]) * r.scale, base, rem);
        if (b >= kBins - 1) continue;  // the last bin is what the others leave
        atomicAdd(&s_count[b], 1u);
        if (r.weigh) atomicAdd(&s_weight[b], weight_int(weight_of(b, rem, s_roots), p.weight_exp));
      }
    }
  }
  const u64 best = wave_max_u64(best_key ? order_word(best_key, best_index) : 0);
  if (lane == 0) s_best[wave] = best;
  if (tokens) atomicAdd(&s_tokens, tokens);
  __syncthreads();
  const int64_t at = (int64_t)row * p.chunks + chunk;
  if (tid == 0) {
    ChunkHead h;
    h.best = 0;
    for (int w = 0; w < kScanWaves; ++w) h.best = s_best[w] > h.best ? s_best[w] : h.best;
    h.base = base;
    h.tokens = s_tokens;
    h.pad[0] = h.pad[1] = h.pad[2] = 0;
    p.heads[at] = h;
  }
  if (r.greedy) return;
#pragma unroll
  for (int b = 0; b < kBins / kScanThreads; ++b) {
    const int i = tid + b * kScanThreads;
    p.counts[at * kBins + i] = s_count[i];
    if (r.weigh) p.weights[at * kBins + i] = s_weight[i];
  }
}

// ---- pick ----
struct PickShared {
  uint32_t count[kBins];  // tokens in bins 0 .. b
  u64 weight[kBins];      // their weight
  union {
    struct {
      u64 word[kList];
      u64 sum[kList];  // weight of entries 0 .. i
    } list;
    struct {
      uint32_t count[kSub];
      u64 weight[kSub];
    } sub;
  };
  double roots[16];
  u64 part[2 * kPickWaves];
  u64 red[4];
  uint32_t n;
};

// A border in the row's order: the token at it, and the tokens and weight up to it, itself included.
struct Border {
  u64 word;
  u64 tokens;
  u64 weight;
};

template <int DT>
struct Pick {
  const SampleParams& p;
  const RowParams& r;
  const Row<DT> x;
  const uint32_t* seg_max;
  PickShared& s;
  double base;
  int tid, wave, lane;

  __device__ Pick(const SampleParams& p_, const RowParams& r_, int row, PickShared& s_)
      : p(p_), r(r_), x(p_, row), seg_max(p_.seg_max + (int64_t)row * p_.segs), s(s_), base(0) {
    tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    lane = tid % kWave;
  }

  // fn(key, index) for every token of the row with key >= least, in no order; segments
  // without one are not read.
  template <typename F>
  __device__ __forceinline__ void each(uint32_t least, F fn) const {
    constexpr int E = kVec<DT>;
    constexpr int kAhead = 4;
    const int segs = (x.vecs + kWave - 1) / kWave;
    for (int s0 = wave * kAhead; s0 < segs; s0 += kPickWaves * kAhead) {
      u32x4 raw[kAhead];
      bool whole[kAhead], want[kAhead];
      uint32_t most[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) most[j] = s0 + j < segs ? seg_max[s0 + j] : 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        want[j] = most[j] != 0 && most[j] >= least;
        whole[j] = false;
        if (want[j]) raw[j] = x.raw((s0 + j) * kWave + lane, whole[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int v = (s0 + j) * kWave + lane;
        if (!want[j] || v >= x.vecs) continue;
        float val[E];
        x.values(v, raw[j], whole[j], val);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t k = key_of(val[e]);
          if (k != 0 && k >= least) fn(k, (uint32_t)(v * E + e - x.skew));
        }
      }
    }
  }

  __device__ __forceinline__ int bin(uint32_t key) const {
    double rem;
    return min(bin_of(finite(logit_of(key)) * r.scale, base, rem), kBins - 1);
  }
  __device__ __forceinline__ u64 weight(uint32_t key) const { return weight_of_key(key, r, base, p.weight_exp, s.roots); }

  // Inclusive sums over the threads, in thread order, of two values at once.
  __device__ void block_scan(u64& a, u64& b) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const u64 y = __shfl_up(a, o), z = __shfl_up(b, o);
      if (lane >= o) {
        a += y;
        b += z;
      }
    }
    __syncthreads();
    if (lane == kWave - 1) {
      s.part[wave] = a;
      s.part[kPickWaves + wave] = b;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      a += s.part[w];
      b += s.part[kPickWaves + w];
    }
  }

  // First bin (of `bins` inclusive sums) whose sum reaches target; the last if none does.
  template <typename T>
  __device__ static int first_reaching(const T* sums, int bins, u64 target) {
    int lo = 0, hi = bins - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if ((u64)sums[mid] >= target)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  }

  // Tokens with key in [klo, khi] and bin in [blo, bhi], in order of the row, with running weights.
  // The caller knows that at most kList qualify.
  __device__ int gather(uint32_t klo, uint32_t khi, int blo, int bhi, uint32_t ilo = 0, uint32_t ihi = 0xFFFFFFFFu) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each(klo, [&](uint32_t k, uint32_t i) {
      if (k > khi || i < ilo || i > ihi) return;
      const int b = bin(k);
      if (b < blo || b > bhi) return;
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kList) s.list.word[at] = order_word(k, i);
    });
    __syncthreads();
    const int n = min((int)s.n, kList);
    int size = kWave;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kPickThreads) s.list.word[i] = 0;
    __syncthreads();
    // bitonic, largest first
    for (int k = 2; k <= size; k <<= 1) {
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int t = tid; t < size / 2; t += kPickThreads) {
          const int a = 2 * t - (t & (j - 1));
          const u64 u = s.list.word[a], v = s.list.word[a + j];
          if (((a & k) == 0) ? u < v : u > v) {
            s.list.word[a] = v;
            s.list.word[a + j] = u;
          }
        }
        __syncthreads();
      }
    }
    // running weights: each thread a run of consecutive entries
    const int per = (n + kPickThreads - 1) / kPickThreads;
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    u64 mine = 0, none = 0;
    for (int i = i0; i < i1; ++i) {
      mine += weight(word_key(s.list.word[i]));
      s.list.sum[i] = mine;
    }
    u64 incl = mine;
    block_scan(incl, none);
    for (int i = i0; i < i1; ++i) s.list.sum[i] += incl - mine;
    __syncthreads();
    return n;
  }

  // The border in bin b at which the running count (by_count) or weight first reaches
  // target; before: what lies in front of the bin.
  __device__ Border border(int b, bool by_count, u64 target) {
    u64 count0 = b > 0 ? s.count[b - 1] : 0, weight0 = b > 0 ? s.weight[b - 1] : 0;
    u64 n = s.count[b] - count0;
    uint32_t klo = 1, khi = 0xFFFFFFFFu;
    bool first = true;
    while (n > (u64)kList) {  // too many to sort: narrow by key
      if (first) {  // the bin's own smallest and largest key
        u64 lo = 0xFFFFFFFFu, hi = 0;
        each(1, [&](uint32_t k, uint32_t) {
          if (bin(k) != b) return;
          lo = k < lo ? k : lo;
          hi = k > hi ? k : hi;
        });
        lo = 0xFFFFFFFFu - wave_max_u64(0xFFFFFFFFu - lo);
        hi = wave_max_u64(hi);
        __syncthreads();
        if (lane == 0) {
          s.part[wave] = lo;
          s.part[kPickWaves + wave] = hi;
        }
        __syncthreads();
        for (int w = 0; w < kPickWaves; ++w) {
          lo = s.part[w] < lo ? s.part[w] : lo;
          hi = s.part[kPickWaves + w] > hi ? s.part[kPickWaves + w] : hi;
        }
        klo = (uint32_t)lo;
        khi = (uint32_t)hi;
        first = false;
      }
      if (klo >= khi) break;
      int shift = 0;
      while (((khi - klo) >> shift) >= kSub) ++shift;
      narrow([&](uint32_t k, uint32_t) { return k >= klo && k <= khi && bin(k) == b ? (int)((khi - k) >> shift) : -1; }, klo);
      // (the histogram's sums may differ from these tokens' in the last place: a weight past them is their end)
      const u64 most = s.sub.weight[kSub - 1], want = target - weight0;
      const int c = by_count ? first_reaching(s.sub.count, kSub, target - count0)
                             : first_reaching(s.sub.weight, kSub, want < most ? want : most);
      const u64 had = c > 0 ? s.sub.count[c - 1] : 0;
      n = s.sub.count[c] - had;
      count0 += had;
      weight0 += c > 0 ? s.sub.weight[c - 1] : 0;
      const uint32_t top = khi - ((uint32_t)c << shift);
      klo = max(klo, top - ((1u << shift) - 1u));
      khi = top;
      __syncthreads();
    }
    uint32_t ilo = 0, ihi = 0xFFFFFFFFu;
    if (n > (u64)kList) {  // one logit: find the token by its index
      const u64 w = weight(klo);
      u64 rank = by_count ? target - count0 - 1 : (w ? (target - weight0 + w - 1) / w - 1 : 0);
      if (rank >= n) rank = n - 1;
      int shift = 0;
      while (((uint32_t)(p.vocab - 1) >> shift) >= kSub) ++shift;
      narrow([&](uint32_t k, uint32_t i) { return k == klo ? (int)(i >> shift) : -1; }, klo);
      const int c = first_reaching(s.sub.count, kSub, rank + 1);
      const u64 had = c > 0 ? s.sub.count[c - 1] : 0;
      count0 += had;
      weight0 += had * w;
      ilo = (uint32_t)c << shift;
      ihi = ilo + (1u << shift) - 1u;
      if (!by_count) target = weight0 + (rank - had + 1) * w;  // the token of that rank, whatever w
      else
        target = count0 + (rank - had) + 1;
      __syncthreads();
    }
    const int m = gather(klo, khi, b, b, ilo, ihi);
    const u64 want = by_count ? target - count0 : target - weight0;
    int i = by_count ? (int)(want < (u64)m ? want : (u64)m) - 1 : first_reaching(s.list.sum, m, want);
    i = max(i, 0);
    const Border out = {s.list.word[i], count0 + i + 1, weight0 + s.list.sum[i]};
    __syncthreads();
    return out;
  }

  // Inclusive counts and weights of the tokens by bucket (which(key, index), -1: none).
  template <typename F>
  __device__ void narrow(F which, uint32_t least) {
    __syncthreads();
    for (int i = tid; i < kSub; i += kPickThreads) {
      s.sub.count[i] = 0;
      s.sub.weight[i] = 0;
    }
    __syncthreads();
    each(least, [&](uint32_t k, uint32_t i) {
      const int c = which(k, i);
      if (c < 0) return;
      atomicAdd(&s.sub.count[c], 1u);
      atomicAdd(&s.sub.weight[c], weight(k));
    });
    __syncthreads();
    constexpr int per = kSub / kPickThreads;
    u64 a = 0, b = 0;
    for (int i = 0; i < per; ++i) {
      a += s.sub.count[tid * per + i];
      b += s.sub.weight[tid * per + i];
    }
    u64 sa = a, sb = b;
    block_scan(sa, sb);
    sa -= a;
    sb -= b;
    for (int i = 0; i < per; ++i) {
      sa += s.sub.count[tid * per + i];
      sb += s.sub.weight[tid * per + i];
      s.sub.count[tid * per + i] = (uint32_t)sa;
      s.sub.weight[tid * per + i] = sb;
    }
    __syncthreads();
  }
};

// f * sum rounded down, or up; exact (equal weights make borders that a rounded product would
// miss).  f > 0, f < 1: m 2^-k with a 24-bit m.
__device__ __forceinline__ u64 share_of(float f, u64 sum, bool up) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, f);
  const uint32_t e = bits >> 23;
  const u64 m = e ? (bits & 0x7FFFFFu) | 0x800000u : bits & 0x7FFFFFu;
  const int k = 150 - (int)max(e, 1u);  // 24 .. 149
  const u64 hi = __umul64hi(sum, m), lo = sum * m;
  u64 whole, rest;  // of the 88-bit product over 2^k
  if (k < 64) {
    whole = (hi << (64 - k)) | (lo >> k);
    rest = lo & ((1ull << k) - 1);
  } else {
    whole = k < 128 ? hi >> (k - 64) : 0;
    rest = lo | (k < 128 ? hi & ((1ull << (k - 64)) - 1) : hi);
  }
  return whole + (up && rest != 0);
}
// floor(u * sum), below sum
__device__ __forceinline__ u64 draw_at(float u, u64 sum) {
  if (!(u > 0.f)) return 0;
  return u < 1.f ? share_of(u, sum, false) : sum - 1;
}
// ceil(top_p * sum), 1 .. sum: the least integer weight that reaches it (top_p < 1)
__device__ __forceinline__ u64 reach_at(float top_p, u64 sum) {
  if (!(top_p > 0.f)) return 1;
  const u64 i = share_of(top_p, sum, true);
  return i > 1 ? i : 1;
}

template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  PickShared& s = *(PickShared*)smem;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const RowParams r = row_params(p, row);
  Pick<DT> k(p, r, row, s);
  const ChunkHead* heads = p.heads + (int64_t)row * p.chunks;
  u64 best = 0;
  double base = -INFINITY;
  u64 tokens = 0;
  for (int c = 0; c < p.chunks; ++c) {
    const ChunkHead h = heads[c];
    best = h.best > best ? h.best : best;
    if (h.tokens) base = fmax(base, h.base);
    tokens += h.tokens;
  }
  RowResult out;
  out.last = best;
  out.base = base;
  out.sum = 1.0;
  out.scale = r.greedy ? -1.0 : r.scale;
  if (best == 0 || r.greedy) {
    if (tid == 0) {
      p.tokens[row] = best ? (int32_t)word_index(best) : -1;
      p.results[row] = out;
    }
    return;
  }
  k.base = base;
  if (tid < 16) s.roots[tid] = kRoots[tid];
  // ---- the row's histogram, as sums from the first bin on ----
  constexpr int per = kBins / kPickThreads;
  u64 count[per], weight[per], ca = 0, wa = 0;
#pragma unroll
  for (int i = 0; i < per; ++i) count[i] = weight[i] = 0;
  for (int c = 0; c < p.chunks; ++c) {
    if (heads[c].tokens == 0) continue;
    const int down = (int)fmin(base - heads[c].base, 64.0);
    const int64_t at = ((int64_t)row * p.chunks + c) * kBins;
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int from = tid * per + i - kBinsPerLog2 * down;
      if (from < 0) continue;
      count[i] += p.counts[at + from];
      if (r.weigh) weight[i] += down < 64 ? p.weights[at + from] >> down : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < per; ++i) {
    ca += count[i];
    wa += weight[i];
  }
  {
    u64 cs = ca, ws = wa;
    k.block_scan(cs, ws);
    cs -= ca;
    ws -= wa;
#pragma unroll
    for (int i = 0; i < per; ++i) {
      cs += count[i];
      ws += weight[i];
      s.count[tid * per + i] = tid * per + i == kBins - 1 ? (uint32_t)tokens : (uint32_t)cs;
      s.weight[tid * per + i] = ws;
    }
  }
  __syncthreads();
  const u64 top_k = r.top_k && (u64)r.top_k < tokens ? r.top_k : tokens;
  const float u = p.uniforms[row];
  const bool cut_p = r.top_p < 1.f;
  const double y_best = finite(logit_of(word_key(best))) * r.scale;
  const double y_min = y_best + kBinsPerLog2 * r.log2_min_p;  // min-p's border in sixteenths of log2
  double rem;
  const int bin_m = r.log2_min_p == -INFINITY ? kBins - 1 : min(bin_of(y_min, base, rem), kBins - 1);
  // ---- the last bin with a kept token, from above ----
  const int bin_k = k.first_reaching(s.count, kBins, top_k);
  int last = bin_k;
  bool weighed = r.weigh;
  if (!weighed && s.count[bin_k] > kList) {
    // a short top-k among many nearly equal logits: the row's weights after all
    weighed = true;
    u64 w[per] = {};
    __syncthreads();
    for (int i = tid; i < kBins; i += kPickThreads) s.weight[i] = 0;
    __syncthreads();
    k.each(1, [&](uint32_t key, uint32_t) {
      const int b = k.bin(key);
      if (b < kBins - 1) atomicAdd(&s.weight[b], k.weight(key));
    });
    __syncthreads();
    u64 a = 0, none = 0;
    for (int i = 0; i < per; ++i) a += w[i] = s.weight[tid * per + i];
    u64 sum = a;
    k.block_scan(sum, none);
    sum -= a;
    for (int i = 0; i < per; ++i) s.weight[tid * per + i] = sum += w[i];
    __syncthreads();
  }
  if (weighed) {
    last = min(last, bin_m);
    if (cut_p) last = min(last, k.first_reaching(s.weight, kBins, reach_at(r.top_p, s.weight[bin_k])));
  }
  if (s.count[last] <= kList) {
    // ---- every token that can be kept, in one sorted list ----
    const int n = k.gather(1, 0xFFFFFFFFu, 0, last);
    // top-p's border is a share of the weight of the first top_k: of the list's, or, where the list
    // ends before them, of the histogram's
    u64 of = 0;
    const int nk = (int)(top_k < (u64)n ? top_k : (u64)n);
    if ((u64)nk == top_k) {
      of = s.list.sum[nk - 1];
    } else if (cut_p) {
      of = top_k == tokens ? s.weight[kBins - 1] : s.weight[bin_k];
      if (top_k != tokens) {
        const Border e = k.border(bin_k, true, top_k);
        of = e.weight;
        k.gather(1, 0xFFFFFFFFu, 0, last);
      }
    }
    const u64 reach = cut_p ? reach_at(r.top_p, of) : ~0ull;
    u64 kept_p = 0, kept_m = 0;
    for (int i = tid; i < nk; i += kPickThreads) {
      const uint32_t key = word_key(s.list.word[i]);
      kept_p += i == 0 || s.list.sum[i - 1] < reach;
      kept_m += finite(logit_of(key)) * r.scale >= y_min;
    }
    k.block_scan(kept_p, kept_m);
    if (tid == kPickThreads - 1) {
      s.red[0] = kept_p;
      s.red[1] = kept_m;
    }
    __syncthreads();
    int kept = (int)min(s.red[0], s.red[1]);
    kept = max(1, min(kept, nk));
    const u64 sum = s.list.sum[kept - 1];
    const int at = k.first_reaching(s.list.sum, kept, draw_at(u, sum) + 1);
    if (tid == 0) {
      p.tokens[row] = (int32_t)word_index(s.list.word[at]);
      out.last = s.list.word[kept - 1];
      out.sum = ldexp((double)sum, -p.weight_exp);
      p.results[row] = out;
    }
    return;
  }
  // ---- a wide nucleus: each border in its own bin ----
  Border end;
  end.word = 1;  // every token
  end.weight = s.weight[kBins - 1];
  if (top_k < tokens) end = k.border(bin_k, true, top_k);
  if (cut_p) {
    const u64 reach = reach_at(r.top_p, end.weight);
    const int b = k.first_reaching(s.weight, kBins, reach);
    const Border e = k.border(b, false, reach);
    if (e.word > end.word) end = e;
  }
  if (r.log2_min_p != -INFINITY && (bin_m > 0 ? s.weight[bin_m - 1] : 0) < end.weight) {
    // tokens of bin_m on the kept side of min-p's border, and the smallest of their order words
    u64 n = 0, w = 0, lo = ~0ull;
    k.each(1, [&](uint32_t key, uint32_t i) {
      if (k.bin(key) != bin_m || !(finite(logit_of(key)) * r.scale >= y_min)) return;
      ++n;
      w += k.weight(key);
      const u64 o = order_word(key, i);
      lo = o < lo ? o : lo;
    });
    lo = ~wave_max_u64(~lo);
    k.block_scan(n, w);
    if (tid == kPickThreads - 1) {
      s.red[0] = n;
      s.red[1] = w;
    }
    __syncthreads();
    if (k.lane == 0) s.part[k.wave] = lo;
    __syncthreads();
    for (int i = 0; i < kPickWaves; ++i) lo = s.part[i] < lo ? s.part[i] : lo;
    const u64 sum = (bin_m > 0 ? s.weight[bin_m - 1] : 0) + s.red[1];
    __syncthreads();
    if (s.red[0] == 0) {
      // the border lies above every token of its bin: the last kept token is the last one before the bin
      if (bin_m > 0 && s.count[bin_m - 1] > 0) {
        const u64 before = s.count[bin_m - 1];
        const Border e = k.border(k.first_reaching(s.count, kBins, before), true, before);
        if (e.word > end.word) end = e;
      }
    } else if (lo > end.word) {
      end.word = lo;
      end.weight = sum;
    }
  }
  const u64 t = draw_at(u, end.weight) + 1;
  const Border d = k.border(k.first_reaching(s.weight, kBins, t), false, t);
  if (tid == 0) {
    // sums of a bin's tokens and of the histogram may differ in the last place
    p.tokens[row] = (int32_t)word_index(d.word > end.word ? d.word : (end.word > 1 ? end.word : d.word));
    out.last = end.word;
    out.sum = ldexp((double)end.weight, -p.weight_exp);
    p.results[row] = out;
  }
}

// ---- probs ----
constexpr int kProbsThreads = 256;
constexpr int kProbsPer = 2;  // vectors per thread

template <int DT>
__global__ __launch_bounds__(kProbsThreads) void sample_probs_kernel(SampleParams p, int groups) {
  constexpr int E = kVec<DT>;
  __shared__ double s_roots[16];
  const int row = blockIdx.x / groups;
  const int v0 = (blockIdx.x % groups) * kProbsThreads * kProbsPer + threadIdx.x;
  if (threadIdx.x < 16) s_roots[threadIdx.x] = kRoots[threadIdx.x];
  __syncthreads();
  const Row<DT> x(p, row);
  const RowResult r = p.results[row];
  const double inv = 1.0 / r.sum;
  float* to = p.probs + (int64_t)row * p.ld_probs;
  u32x4 raw[kProbsPer];
  bool whole[kProbsPer];
#pragma unroll
  for (int j = 0; j < kProbsPer; ++j) {
    whole[j] = false;
    if (v0 + j * kProbsThreads < x.vecs) raw[j] = x.raw(v0 + j * kProbsThreads, whole[j]);
  }
#pragma unroll
  for (int j = 0; j < kProbsPer; ++j) {
    const int v = v0 + j * kProbsThreads;
    if (v >= x.vecs) continue;
    float val[E], out[E];
    x.values(v, raw[j], whole[j], val);
    const int t0 = v * E - x.skew;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      out[e] = 0.f;
      const uint32_t key = key_of(val[e]);
      if (key == 0 || r.last == 0 || order_word(key, t0 + e) < r.last) continue;
      if (r.scale < 0.0) {
        out[e] = 1.f;
      } else {
        double rem;
        const int b = bin_of(finite(val[e]) * r.scale, r.base, rem);
        out[e] = (float)(weight_of(b, rem, s_roots) * inv);
      }
    }
    if (whole[j] && ((uintptr_t)(to + t0) & 15) == 0) {
#pragma unroll
      for (int e = 0; e < E; e += 4) *(floatx4*)(to + t0 + e) = floatx4{out[e], out[e + 1], out[e + 2], out[e + 3]};
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (t0 + e >= 0 && t0 + e < x.vocab) to[t0 + e] = out[e];
    }
  }
}

// ---- host ----
int elements_per_vec(int dtype) { return dtype == NE_DTYPE_FP32 ? 4 : 8; }

// Chunks of a row: enough work-groups to fill the chip twice, at least one iteration of the scan each.
int row_chunks(int rows, int segs) {
  const int want = ceil_div(2 * kNumCu, rows < 1 ? 1 : rows);
  const int most = ceil_div(segs, kScanWaves * kScanSegs);
  return want < most ? want : most;
}

struct Layout {
  int chunks, segs;
  size_t heads, counts, weights, seg_max, results, bytes;
};
Layout layout_of(int rows, int vocab, int dtype) {
  Layout l;
  const int e = elements_per_vec(dtype);
  rows = rows < kRowBatch ? rows : kRowBatch;
  l.segs = ceil_div(vocab + e - 1, e * kWave);  // a row off the 16-byte grid may touch one vector more
  l.chunks = row_chunks(rows, l.segs);
  const size_t n = (size_t)rows * l.chunks;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.heads = take(n * sizeof(ChunkHead));
  l.weights = take(n * kBins * sizeof(u64));
  l.counts = take(n * kBins * sizeof(uint32_t));
  l.seg_max = take((size_t)rows * l.segs * sizeof(uint32_t));
  l.results = take((size_t)rows * sizeof(RowResult));
  l.bytes = at;
  return l;
}

template <int DT>
int launch(const SampleParams& p, hipStream_t s) {
  hipLaunchKernelGGL(sample_scan_kernel<DT>, dim3(p.rows * p.chunks), dim3(kScanThreads), 0, s, p);
  int rc = check_launch("sample_scan");
  if (rc != NE_OK) return rc;
  static const hipError_t attr = hipFuncSetAttribute((const void*)sample_pick_kernel<DT>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(PickShared));
  if (attr != hipSuccess) {
    set_error("sample_pick: cannot reserve %d bytes of LDS: %s", (int)sizeof(PickShared), hipGetErrorString(attr));
    return NE_ELAUNCH;
  }
  hipLaunchKernelGGL(sample_pick_kernel<DT>, dim3(p.rows), dim3(kPickThreads), sizeof(PickShared), s, p);
  rc = check_launch("sample_pick");
  if (rc != NE_OK || !p.probs) return rc;
  const int vecs = ceil_div(p.vocab + kVec<DT> - 1, kVec<DT>);
  const int groups = ceil_div(vecs, kProbsThreads * kProbsPer);
  hipLaunchKernelGGL(sample_probs_kernel<DT>, dim3(p.rows * groups), dim3(kProbsThreads), 0, s, p, groups);
  return check_launch("sample_probs");
}

}  // namespace

}  // namespace ne

extern "C" size_t ne_sample_workspace_size(int32_t rows, int32_t vocab, int32_t dtype) {
  if (rows < 1 || vocab < 1 || vocab > ne::kMaxVocab || dtype < NE_DTYPE_BF16 || dtype > NE_DTYPE_FP32) return 0;
  return ne::layout_of(rows, vocab, dtype).bytes;
}

extern "C" int ne_sample(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t vocab,
                         const float* uniforms, const float* temperatures, float temperature, const int32_t* top_ks,
                         int32_t top_k, const float* top_ps, float top_p, const float* min_ps, float min_p,
                         int32_t* tokens, float* probs, int64_t ld_probs, void* workspace, size_t workspace_bytes,
                         void* stream) {
  using namespace ne;
  NE_CHECK_ARG(rows >= 0 && vocab >= 1, "bad sizes: %d rows of %d", rows, vocab);
  NE_CHECK_ARG(dtype == NE_DTYPE_BF16 || dtype == NE_DTYPE_FP16 || dtype == NE_DTYPE_FP32,
               "logits must be bf16, fp16 or fp32");
  NE_CHECK_SUPPORTED(vocab <= kMaxVocab, "vocab %d exceeds %d", vocab, kMaxVocab);
  if (rows == 0) return NE_OK;
  NE_CHECK_ARG(logits && uniforms && tokens && workspace, "null pointer argument");
  NE_CHECK_ARG(ld >= vocab || rows == 1, "row stride %lld below %d", (long long)ld, vocab);
  NE_CHECK_ARG(!probs || ld_probs >= vocab || rows == 1, "probs row stride %lld below %d", (long long)ld_probs, vocab);
  NE_CHECK_ARG(temperatures || (temperature >= 0.f && temperature < INFINITY), "temperature must be finite and >= 0");
  NE_CHECK_ARG(top_ps || top_p == top_p, "top_p is NaN");
  NE_CHECK_ARG(min_ps || min_p == min_p, "min_p is NaN");
  NE_CHECK_ARG((uintptr_t)logits % (dtype == NE_DTYPE_FP32 ? 4 : 2) == 0, "logits off their elements' alignment");
  const Layout l = layout_of(rows, vocab, dtype);
  if (workspace_bytes < l.bytes) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, l.bytes);
    return NE_EWORKSPACE;
  }
  NE_CHECK_ARG((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  char* ws = (char*)workspace;
  SampleParams p;
  memset(&p, 0, sizeof(p));
  p.vocab = vocab;
  p.ld = ld;
  p.chunks = l.chunks;
  p.segs = l.segs;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.ld_probs = ld_probs;
  p.heads = (ChunkHead*)(ws + l.heads);
  p.counts = (uint32_t*)(ws + l.counts);
  p.weights = (u64*)(ws + l.weights);
  p.seg_max = (uint32_t*)(ws + l.seg_max);
  p.results = (RowResult*)(ws + l.results);
  p.weight_exp = 63;
  for (int v = 1; v < vocab; v *= 2) --p.weight_exp;
  if (p.weight_exp > 51) p.weight_exp = 51;
  const int esz = dtype == NE_DTYPE_FP32 ? 4 : 2;
  for (int r0 = 0; r0 < rows; r0 += kRowBatch) {  // batches share the workspace in stream order
    p.rows = rows - r0 < kRowBatch ? rows - r0 : kRowBatch;
    p.logits = (const char*)logits + (int64_t)r0 * ld * esz;
    p.uniforms = uniforms + r0;
    p.temperatures = temperatures ? temperatures + r0 : nullptr;
    p.top_ks = top_ks ? top_ks + r0 : nullptr;
    p.top_ps = top_ps ? top_ps + r0 : nullptr;
    p.min_ps = min_ps ? min_ps + r0 : nullptr;
    p.tokens = tokens + r0;
    p.probs = probs ? probs + (int64_t)r0 * ld_probs : nullptr;
    const int rc = dtype == NE_DTYPE_BF16   ? launch<NE_DTYPE_BF16>(p, (hipStream_t)stream)
                   : dtype == NE_DTYPE_FP16 ? launch<NE_DTYPE_FP16>(p, (hipStream_t)stream)
                                            : launch<NE_DTYPE_FP32>(p, (hipStream_t)stream);
    if (rc != NE_OK) return rc;
  }
  return NE_OK;
}
