// Sampling a token per row of logits from a given uniform, under temperature, top-k,
// top-p and min-p, and the filtered distribution itself.
//
// Definition.  A row's tokens are ordered by logit (descending), then by index
// (ascending); NaN and -inf are no tokens.  y = x log2(e) / T; a token's weight is
// 2^(y - Y) with one Y per row.  Kept: the first n = min(n_k, n_p, n_m) tokens of the order,
//   n_k = top_k (all, where top_k is 0 or less),
//   n_p = the fewest whose weight reaches top_p times the weight of the first n_k
//         (all, where top_p is 1 or more),
//   n_m = the tokens with weight at least min_p times the largest (above 1: none),
// and at least one.  The token drawn is the first whose running weight exceeds
// u * (kept weight).  T = 0 keeps the first token alone.
//
// Weights are integers, rint(2^(y - Y) * 2^S) with 2^S * vocab <= 2^63, computed in 64-bit
// floating point: a sum of them does not depend on its order (nor on that of atomics), so a call
// repeated gives the same bits.  The split of a row into chunks does count.  A chunk weighs its
// tokens relative to its own largest logit, and histograms brought to the row's drop up to a unit
// of 2^-S per bin and chunk (fp32: and each time a chunk's largest logit rises).  Chunks follow
// the number of rows, so a row may place a border that much apart in a batch of another size.
// With the tokens' own rounding a border between two tokens is off by at most ~2^-S of the row's
// largest weight per token, and per bin and chunk (S = 45 for 151,936 tokens, 3 to 7 chunks in 16
// bits, up to 38 in fp32, 736 bins of any weight): a draw in the tail, whose tokens weigh 1e-11 of
// the largest, may fall on a neighbour, one in 1e6 of a peaked row's.  32-bit weights would move every
// border of a flat row by 1e-7, a wrong token in a hundred rows of 100,000 tokens.
//
// Three kernels.
//   scan   rows x chunks: reads the logits once.  Per 128-byte segment the largest key; per
//          chunk the largest and its vector, and a histogram over y in steps of 1/16 (1,024
//          bins below the chunk's own base Y, counts and, unless top-k is short, weights).
//          The base is an integer, so histograms of unlike bases merge by shifting 16 bins
//          and one bit per step.  16-bit logits are counted by value first, and each value
//          is weighed once; fp32 ones are weighed one by one.
//   pick   one work-group per row: merges the row's histograms, finds the last bin that can
//          hold a kept token, and, where at most 4,096 tokens lie above its end, gathers
//          them (only from segments whose largest key reaches it), sorts them in LDS and
//          finishes there.  A wide nucleus is handled bin by bin: the border of each filter
//          and the draw lie in one bin each, whose tokens are gathered and sorted; a bin
//          with more tokens than the list holds is narrowed by key first, and a run of
//          equal logits by index.
//   probs  rows x chunks: kept weight / sum per token, if asked for.
// What bounds it, at 151,936 tokens a row.  320 rows (bf16, top-p, with probabilities) 152 us:
// the scan 42, for its ~10 operations per element and the weights of ~3,000 values per chunk
// (67% of the vector units' time); pick 46, rows' chains of passes (the longest 40) in two rounds of
// work-groups, one per CU for its 103 KB of LDS and 1,024 threads of 128 registers; probs 43, its
// bytes (292 MB, 6.9 TB/s).  64 rows 41 us: 11 and 24.  One row 29 us: 6 and 19, a chain of round
// trips through memory and barriers.  200 rows of 32,003 (fp32) 48 us: 22, for 65 vector operations
// per element (half of it) and the sums in LDS, and 24.
#include <math.h>
#include <string.h>

#include <type_traits>

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
constexpr int kScanLines = 2;         // lines (of a vector per lane) per wave and iteration
constexpr int kSegVecs = 8;           // vectors of a segment
constexpr int kLineSegs = kWave / kSegVecs;
constexpr int kCountThreads = 1024;
constexpr int kCountWaves = kCountThreads / kWave;
constexpr int kCountLines = 4;
constexpr int kCountLeast = 3 * kCountWaves;
constexpr int kCountMost = 127;       // lines of a chunk: 65,024 elements, whose counts fit 16 bits
constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / kWave;
constexpr int kList = 4096;           // tokens that pick sorts in LDS
constexpr int kShortTopK = 1024;      // up to here the scan counts tokens and leaves their weights to pick
constexpr int kSub = 2048;            // buckets of a narrowing pass
constexpr int kSortBuckets = 2048;    // and of a sort
constexpr int kSegsHeld = 4096;       // segments' largest keys that pick keeps in LDS
constexpr int kRankMost = 64;         // tokens of a bucket that are ranked
constexpr int kMaxVocab = 1 << 20;
constexpr int kRowBatch = 1024;       // rows per launch: bounds the workspace

// One chunk's result; its histogram follows in arrays of their own.
struct ChunkHead {
  u64 best;     // largest key and its first vector (key, ~vector); 0: no token
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
constexpr uint32_t kLeastKey = 0x00800000u;  // of the largest negative number
constexpr uint32_t kNegativeZero = 0x7FFFFFFFu;  // below +0's key, and no token's, as -0 has +0's
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
  const u32x4* base;   // vector 0: a scalar load of a vector needs its base on the grid too
  const u32x4* whole;  // the first vector that lies in the row, or some memory where none does
  int skew, vocab, vecs;
  int whole0, wholes;  // vectors that lie in the row
  __device__ Row(const SampleParams& p, int row) {
    constexpr int kEsz = 16 / kVec<DT>;
    const char* at = (const char*)p.logits + (int64_t)row * p.ld * kEsz;
    skew = (int)((uintptr_t)at & 15) / kEsz;
    base = (const u32x4*)(at - skew * kEsz);
    vocab = p.vocab;
    vecs = (vocab + skew + kVec<DT> - 1) / kVec<DT>;
    whole0 = skew > 0;
    wholes = max((vocab + skew) / kVec<DT> - whole0, 0);
    whole = wholes > 0 ? base + whole0 : (const u32x4*)p.heads;
  }
  __device__ __forceinline__ bool is_whole(int v) const { return (uint32_t)(v - whole0) < (uint32_t)wholes; }
  // All of a line (a vector per lane) lies in the row.
  __device__ __forceinline__ bool inner(int line) const { return line * kWave >= whole0 && (line + 1) * kWave <= whole0 + wholes; }
  // Vector v where that lies in the row, else another: a load without a branch, so that those after it need
  // not be waited for.
  __device__ __forceinline__ u32x4 ahead(int v) const { return whole[min(max(v - whole0, 0), max(wholes - 1, 0))]; }
  // Vector v, NaN for what lies outside the row.
  __device__ __forceinline__ u32x4 vec(int v) const {
    const int t0 = v * kVec<DT> - skew;
    if (is_whole(v)) return base[v];
    const uint32_t none = DT == NE_DTYPE_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    uint32_t out[4] = {none, none, none, none};
    if (v >= vecs) return u32x4{none, none, none, none};
#pragma unroll 1
    for (int e = 0; e < kVec<DT>; ++e) {
      if (t0 + e < 0 || t0 + e >= vocab) continue;
      uint32_t bits, keep = 0;
      if constexpr (DT == NE_DTYPE_FP32) {
        bits = ((const uint32_t*)(base + v))[e];
      } else {
        bits = (uint32_t)((const uint16_t*)(base + v))[e] << (16 * (e & 1));
        keep = e & 1 ? 0xFFFFu : 0xFFFF0000u;
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) out[d] = d == e * 4 / kVec<DT> ? (out[d] & keep) | bits : out[d];
    }
    return u32x4{out[0], out[1], out[2], out[3]};
  }
};
// Element e of a dword's one or two.
template <int DT>
__device__ __forceinline__ float element(uint32_t d, int e) {
  if (DT == NE_DTYPE_FP32) return __builtin_bit_cast(float, d);
  const uint16_t h = (uint16_t)(d >> (16 * e));
  return DT == NE_DTYPE_FP16 ? f16_to_f32(h) : bf16_to_f32(h);
}
template <int DT>
__device__ __forceinline__ void values(u32x4 x, float (&out)[kVec<DT>]) {
#pragma unroll
  for (int e = 0; e < kVec<DT>; ++e) {
    const uint32_t d = x[e * 4 / kVec<DT>];  // (a bit cast of the vector's element itself reads element 0)
    out[e] = element<DT>(d, e % (kVec<DT> / 4));
  }
}

// ---- row parameters ----
struct RowParams {
  double scale;  // 16 log2(e) / T
  float top_p, min_p;
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
  if (m > 1.f && p.vocab > 1) r.top_k = 1;  // no token weighs more than the first: it alone is kept
  r.weigh = !r.greedy && (r.top_k == 0 || r.top_k > kShortTopK);
  r.min_p = m;
  return r;
}

// ---- weights ----
// y in sixteenths is split into its floor f (a bin) and a remainder r in [0, 1):
// 2^(y - Y) = 2^((f - 16 Y) / 16) * 2^(r / 16); floor and remainder are exact, so a
// token's bin is the same under every base.  Table: 2^(j / 16 + 1 / 32), j = 0..15.
__constant__ const double kRoots[16] = {
    1.0218971486541166, 1.0671404006768237, 1.1143867425958924, 1.1637248587775775, 1.215247359980469,
    1.2690509571917332, 1.3252366431597413, 1.383909881963832, 1.4451808069770467, 1.5091644275934228,
    1.5759808451078865, 1.645755478153965, 1.718619298122478, 1.7947090750031072, 1.8741676341103,
    1.9571441241754002};

// The token's bin below base16 = 16 Y (0 = largest y) and its remainder; base16 > 16 y, up to the
// rounding of values past 2^53 (a temperature next to 0), which the lower bound catches.
__device__ __forceinline__ int bin_of(double y16, double base16, double& rem) {
  const double f = floor(y16);
  rem = y16 - f;
  // past kBins - 1: too small to weigh
  return max((int)fmin(base16 - f, (double)(1 << 20)), 1) - 1;
}
// 2^(y - Y + s) for a token of bin b and remainder rem, above 2^-1000.  2^(rem / 16 - 1 / 32) by its
// series in t = rem - 1/2, coefficients (ln 2 / 16)^k / k!: |t ln 2 / 16| < 0.0217, whose seventh
// power over 7! is 4.5e-16.  The exponent is added to the bits.
__device__ __forceinline__ double weight_of(int b, double rem, int s, const double* roots) {
  constexpr double L = 0.6931471805599453 / kBinsPerLog2;
  const int q = b + 1;
  const double t = rem - 0.5;
  double e = L * L * L * L * L * L / 720;
  e = fma(e, t, L * L * L * L * L / 120);
  e = fma(e, t, L * L * L * L / 24);
  e = fma(e, t, L * L * L / 6);
  e = fma(e, t, L * L / 2);
  e = fma(e, t, L);
  e = fma(e, t, 1.0);
  const u64 bits = __builtin_bit_cast(u64, e * roots[-q & 15]);
  const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)(s - ((q + 15) >> 4)) << 20);
  return __builtin_bit_cast(double, ((u64)high << 32) | (uint32_t)bits);
}
// rint of a weight below 2^52: adding 2^52 leaves the integer in the low mantissa bits
__device__ __forceinline__ u64 weight_int(double w) {
  return __builtin_bit_cast(u64, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ u64 weight_of_key(uint32_t key, const RowParams& r, double base16, int s, const double* roots) {
  double rem;
  const int b = bin_of(finite(logit_of(key)) * r.scale, base16, rem);
  return b < kBins ? weight_int(weight_of(b, rem, s, roots)) : 0;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return ((u64)hi << 32) | lo;
}
// Sums over the lanes up to each: within rows of 16 lanes, then over rows.
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
  return ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), kWave - 1) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, kWave - 1);
}
__device__ __forceinline__ u64 max_u64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
  v = max_u64(v, dpp_u64<0x111, 0xF>(v));
  v = max_u64(v, dpp_u64<0x112, 0xF>(v));
  v = max_u64(v, dpp_u64<0x114, 0xF>(v));
  v = max_u64(v, dpp_u64<0x118, 0xF>(v));
  v = max_u64(v, dpp_u64<0x142, 0xA>(v));
  return last_lane(max_u64(v, dpp_u64<0x143, 0xC>(v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
// The maximum over 16 lanes, in the last.
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
  return dpp_max<0x118, 0xF>(dpp_max<0x114, 0xF>(dpp_max<0x112, 0xF>(dpp_max<0x111, 0xF>(v))));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = dpp_max<0x143, 0xC>(dpp_max<0x142, 0xA>(row_max_u32(v)));
  return __builtin_amdgcn_readlane((int)v, kWave - 1);
}
// The maximum over the 8 lanes of a segment, in each.
__device__ __forceinline__ float seg_max_of(float v) {
  auto from = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v = fmaxf(v, from(v, std::integral_constant<int, 0xB1>{}));   // lanes 1 0 3 2
  v = fmaxf(v, from(v, std::integral_constant<int, 0x4E>{}));   // 2 3 0 1
  return fmaxf(v, from(v, std::integral_constant<int, 0x141>{}));  // 7 .. 0 of each 8
}

// Index of the first token of vector v that has this key.
template <int DT>
__device__ __forceinline__ uint32_t index_in(const Row<DT>& x, int v, uint32_t key) {
  float val[kVec<DT>];
  values<DT>(x.vec(v), val);
  int at = kVec<DT> - 1;
#pragma unroll
  for (int e = kVec<DT> - 2; e >= 0; --e) at = key_of(val[e]) == key ? e : at;
  return (uint32_t)(v * kVec<DT> + at - x.skew);
}

// ---- count: the scan of 16-bit logits ----
// A work-group counts its chunk's values by their bits (two counts a word: a value and its negative), and
// weighs each value that occurs once, times its count: integers, so the sum is the tokens' own.  Counted are
// magnitudes in a window, 2^-14 to 2^8 (bf16), 2^-7 to 2^7 (fp16); the few values outside are listed, and a
// chunk of more than the list holds is read again for them.  The window leaves room for two work-groups per
// CU: a table of all values took 53 us for 320 rows of 151,936.
template <int DT>
constexpr uint32_t kWindow = DT == NE_DTYPE_FP16 ? 14 * 1024 : 22 * 128;
template <int DT>
constexpr uint32_t kWindowFrom = DT == NE_DTYPE_FP16 ? (15 - 7) << 10 : (127 - 14) << 7;
constexpr int kListed = 4096;
template <int DT>
constexpr int16_t kInfinity = DT == NE_DTYPE_FP16 ? 0x7C00 : 0x7F80;
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
// Two halves' order as signed integers, and back.  Positive NaN come out above everything.
__device__ __forceinline__ i16x2 order_pair(uint32_t u) {
  const i16x2 h = __builtin_bit_cast(i16x2, u);
  return h ^ ((h >> 15) & (int16_t)0x7FFF);
}
template <int DT>
__device__ __forceinline__ float logit_in_order(int v) { return element<DT>((uint16_t)(v ^ ((v >> 15) & 0x7FFF)), 0); }
__device__ __forceinline__ int seg_max_of(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true));
  return max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true));
}
template <int DT>
struct CountShared {
  uint32_t pair[kWindow<DT> + 4];  // (one more for what is outside)
  u64 weight[kBins];
  uint32_t count[kBins];
  uint16_t listed[kListed];
  double roots[16];
  uint32_t best[kCountWaves];
  uint32_t tokens, outside;
};
template <int DT>
__global__ __launch_bounds__(kCountThreads, 8) void sample_count_kernel(SampleParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  CountShared<DT>& s = *(CountShared<DT>*)smem;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int row = blockIdx.y, chunk = blockIdx.x;
  const RowParams r = row_params(p, row);
  const Row<DT> x(p, row);
  const int lines = (x.vecs + kWave - 1) / kWave;
  const int l0 = (uint32_t)(lines * chunk) / (uint32_t)p.chunks, l1 = (uint32_t)(lines * (chunk + 1)) / (uint32_t)p.chunks;
  u32x4 raw[kCountLines];
#pragma unroll
  for (int j = 0; j < kCountLines; ++j) raw[j] = x.ahead((l0 + wave + j * kCountWaves) * kWave + lane);
  // a token whose magnitude the window does not hold
  auto is_outside = [](uint32_t bits) { return (bits & 0x7FFF) - kWindowFrom<DT> >= kWindow<DT> && element<DT>(bits, 0) > -INFINITY; };
  for (int i = tid; i < (int)(kWindow<DT> / 4) + 1; i += kCountThreads) ((u32x4*)s.pair)[i] = u32x4{0, 0, 0, 0};
  s.weight[tid] = 0;
  s.count[tid] = 0;
  if (tid < 16) s.roots[tid] = kRoots[tid];
  if (tid == 0) s.tokens = s.outside = 0;
  __syncthreads();
  int best_order = INT16_MIN, best_vec = l0 * kWave;
  for (int at = l0 + wave; at < l1; at += kCountLines * kCountWaves) {
    int seg_top = INT16_MIN;  // of line lane % kSegVecs
#pragma unroll
    for (int j = 0; j < kCountLines; ++j) {
      const int line = at + j * kCountWaves;
      if (line >= l1) continue;
      u32x4 now = raw[j];
      raw[j] = x.ahead((line + kCountLines * kCountWaves) * kWave + lane);
      if (!x.inner(line)) now = x.vec(line * kWave + lane);
      i16x2 tops = {INT16_MIN, INT16_MIN};
      uint32_t far = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = now[e];
        // (as byte offsets)
        const uint32_t lo = min(((u & 0x7FFF) << 2) - 4 * kWindowFrom<DT>, 4 * kWindow<DT>);
        const uint32_t hi = min((((u >> 16) & 0x7FFF) << 2) - 4 * kWindowFrom<DT>, 4 * kWindow<DT>);
        far = max(max(far, lo), hi);
        atomicAdd((uint32_t*)((char*)s.pair + lo), (int16_t)u < 0 ? 0x10000u : 1u);
        atomicAdd((uint32_t*)((char*)s.pair + hi), (int32_t)u < 0 ? 0x10000u : 1u);
        tops = __builtin_elementwise_max(tops, order_pair(u));
      }
      int top = max(tops[0], tops[1]);
      if (top > kInfinity<DT>) {  // a NaN among them
        top = INT16_MIN;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const i16x2 h = order_pair(now[e]);
          top = max(top, max(h[0] > kInfinity<DT> ? INT16_MIN : (int)h[0], h[1] > kInfinity<DT> ? INT16_MIN : (int)h[1]));
        }
      }
      top += top == -1;  // -0 is no smaller than +0
      if (far == 4 * kWindow<DT>) {
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint32_t d = e < 4 ? e < 2 ? now[0] : now[1] : e < 6 ? now[2] : now[3];
          const uint32_t bits = d >> (16 * (e & 1)) & 0xFFFF;
          if (!is_outside(bits)) continue;
          const uint32_t to = atomicAdd(&s.outside, 1u);
          if (to < (uint32_t)kListed) s.listed[to] = (uint16_t)bits;
        }
      }
      if (top > best_order) {  // a lane's vectors come in order
        best_order = top;
        best_vec = line * kWave + lane;
      }
      top = seg_max_of(top);
      seg_top = lane % kSegVecs == j ? top : seg_top;
    }
    const int line = at + lane % kSegVecs * kCountWaves;
    if (lane % kSegVecs < kCountLines && line < l1)
      p.seg_max[(int64_t)row * p.segs + line * kLineSegs + lane / kSegVecs] = key_of(logit_in_order<DT>(seg_top));
  }
  // the largest, and its first vector (of at most kCountMost lines)
  const uint32_t mine = wave_max_u32((uint32_t)(best_order - INT16_MIN) << 16 | (0xFFFF - (best_vec - l0 * kWave)));
  if (lane == 0) s.best[wave] = mine;
  __syncthreads();
  const uint32_t word = __builtin_amdgcn_readlane((int)row_max_u32(s.best[lane % kCountWaves]), 15);
  const uint32_t all_key = key_of(logit_in_order<DT>((int)(word >> 16) + INT16_MIN));
  const u64 all = all_key ? order_word(all_key, l0 * kWave + 0xFFFF - (word & 0xFFFF)) : 0;
  const double base = all && !r.greedy ? floor(finite(logit_of(all_key)) * r.scale / kBinsPerLog2) + 1.0 : 0.0;
  uint32_t tokens = 0;
  if (all && !r.greedy) {
    const double base16 = kBinsPerLog2 * base;
    auto add = [&](uint32_t bits, uint32_t n) {
      const float v = element<DT>(bits, 0);
      double rem;
      const int b = bin_of(finite(v) * r.scale, base16, rem);
      const u64 w = weight_int(weight_of(b, rem, p.weight_exp, s.roots));
      tokens += n;
      if (n != 0 && b < kBins - 1) {  // the last bin is what the others leave
        atomicAdd(&s.count[b], n);
        if (r.weigh) atomicAdd(&s.weight[b], n * w);
      }
    };
    for (int i = tid; i < (int)kWindow<DT>; i += kCountThreads) {
      const uint32_t two = s.pair[i];
      if (two == 0) continue;
      add(kWindowFrom<DT> + i, two & 0xFFFF);  // (both at once: a chain of 64-bit operations each)
      add((kWindowFrom<DT> + i) | 0x8000, two >> 16);
    }
    const uint32_t outside = s.outside;
    if (outside <= (uint32_t)kListed) {
      for (int i = tid; i < (int)outside; i += kCountThreads) add(s.listed[i], 1);
    } else {
      for (int line = l0 + wave; line < l1; line += kCountWaves) {
        const u32x4 four = x.vec(line * kWave + lane);
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint32_t d = e < 4 ? e < 2 ? four[0] : four[1] : e < 6 ? four[2] : four[3];
          const uint32_t bits = d >> (16 * (e & 1)) & 0xFFFF;
          if (is_outside(bits)) add(bits, 1);
        }
      }
    }
    const uint32_t sum = (uint32_t)last_lane(wave_scan(tokens));
    if (lane == 0 && sum) atomicAdd(&s.tokens, sum);
  }
  __syncthreads();
  const int64_t to = (int64_t)row * p.chunks + chunk;
  if (tid == 0) {
    ChunkHead h;
    h.best = all;
    h.base = base;
    h.tokens = s.tokens;
    h.pad[0] = h.pad[1] = h.pad[2] = 0;
    p.heads[to] = h;
  }
  if (r.greedy) return;
  p.counts[to * kBins + tid] = s.count[tid];
  if (r.weigh) p.weights[to * kBins + tid] = s.weight[tid];
}

// ---- scan of fp32 logits ----
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(SampleParams p) {
  constexpr int DT = NE_DTYPE_FP32;
  constexpr int E = kVec<DT>;
  __shared__ uint32_t s_count[kBins];
  __shared__ u64 s_weight[kBins];
  __shared__ double s_roots[16];
  __shared__ float s_max[2][kScanWaves];
  __shared__ u64 s_best[kScanWaves];
  __shared__ uint32_t s_tokens;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int row = blockIdx.y, chunk = blockIdx.x;
  const RowParams r = row_params(p, row);
  const Row<DT> x(p, row);
  const int lines = (x.vecs + kWave - 1) / kWave;
  const int l0 = (uint32_t)(lines * chunk) / (uint32_t)p.chunks, l1 = (uint32_t)(lines * (chunk + 1)) / (uint32_t)p.chunks;
  if (tid < 16) s_roots[tid] = kRoots[tid];
  if (tid == 0) s_tokens = 0;
#pragma unroll
  for (int b = 0; b < kBins / kScanThreads; ++b) {
    s_count[tid + b * kScanThreads] = 0;
    s_weight[tid + b * kScanThreads] = 0;
  }
  float best_logit = -INFINITY;
  int best_vec = 0;
  uint32_t tokens = 0;
  double base = 0;
  bool any = false;  // base is set
  constexpr int kStep = kScanWaves * kScanLines;
  u32x4 raw[kScanLines];
  auto load = [&](int s0) {
#pragma unroll
    for (int j = 0; j < kScanLines; ++j) {
      const int line = s0 + wave * kScanLines + j;
      raw[j] = x.ahead(line * kWave + lane);
    }
  };
  load(l0);
  int turn = 0;
  for (int s0 = l0; s0 < l1; s0 += kStep, turn ^= 1) {
    float val[kScanLines][E];
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kScanLines; ++j) {
      const int line = s0 + wave * kScanLines + j;
      const int v = line * kWave + lane;
#pragma unroll
      for (int e = 0; e < E; ++e) val[j][e] = NAN;
      if (line < l1) {
        float here = -INFINITY;
        if (!x.inner(line)) raw[j] = x.vec(v);
        values<DT>(raw[j], val[j]);
#pragma unroll
        for (int e = 0; e < E; ++e) here = fmaxf(here, val[j][e]);  // (not NaN)
        if (here > best_logit) {  // a lane's vectors come in order
          best_logit = here;
          best_vec = v;
        }
        here = seg_max_of(here);
        if (lane % kSegVecs == 0) p.seg_max[(int64_t)row * p.segs + line * kLineSegs + lane / kSegVecs] = key_of(here);
        most = fmaxf(most, here);
      }
    }
    most = wave_max(most);
    if (s0 + kStep < l1) load(s0 + kStep);
    if (lane == 0) s_max[turn][wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) most = fmaxf(most, s_max[turn][w]);
    if (r.greedy || !(most > -INFINITY)) continue;
    const double top = floor(finite(most) * r.scale / kBinsPerLog2) + 1.0;
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
    const double base16 = kBinsPerLog2 * base;
#pragma unroll
    for (int j = 0; j < kScanLines; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool is = val[j][e] > -INFINITY;
        tokens += is;
        double rem;
        const int b = bin_of(finite(val[j][e]) * r.scale, base16, rem);
        if (is && b < kBins - 1) {  // the last bin is what the others leave
          atomicAdd(&s_count[b], 1u);
          if (r.weigh) atomicAdd(&s_weight[b], weight_int(weight_of(b, rem, p.weight_exp, s_roots)));
        }
      }
    }
  }
  const uint32_t best_key = key_of(best_logit);
  const u64 best = wave_max_u64(best_key ? order_word(best_key, best_vec) : 0);
  if (lane == 0) s_best[wave] = best;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) tokens += __shfl_xor((int)tokens, o);
  if (lane == 0 && tokens) atomicAdd(&s_tokens, tokens);
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
      uint32_t count[kSub];  // tokens in buckets 0 .. c
      u64 weight[kSub];
    } sub;
    int down[2 * kNumCu];  // each chunk's base below the row's
  };
  uint32_t bucket[kSortBuckets + 1];
  uint32_t seg[kSegsHeld];  // the first segments' largest keys
  double roots[16];
  u64 part[2 * kPickWaves];
  u64 red[4];
  uint32_t n, wanted;
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
// floor(u * sum), below sum (u < 1)
__device__ __forceinline__ u64 draw_at(float u, u64 sum) { return u > 0.f ? share_of(u, sum, false) : 0; }
// ceil(top_p * sum), 1 .. sum: the least integer weight that reaches it (top_p < 1)
__device__ __forceinline__ u64 reach_at(float top_p, u64 sum) {
  if (!(top_p > 0.f)) return 1;
  const u64 i = share_of(top_p, sum, true);
  return i > 1 ? i : 1;
}

// The work-group's state is the same in every lane: kept in scalar registers.
__device__ __forceinline__ uint32_t uni(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ u64 uni(u64 v) { return ((u64)uni((uint32_t)(v >> 32)) << 32) | uni((uint32_t)v); }
__device__ __forceinline__ double uni(double v) { return __builtin_bit_cast(double, uni(__builtin_bit_cast(u64, v))); }

// First of n inclusive sums that reaches target; the last if none does.  Every lane of a wave takes part:
// a step leaves a 64th of the sums.
template <typename T>
__device__ __forceinline__ int first_reaching(const T* sums, int n, u64 target) {
  const int lane = threadIdx.x % kWave;
  int lo = 0;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave;
    const u64 reach = __ballot((u64)sums[lo + min((lane + 1) * step, n) - 1] >= target);
    const int f = reach ? (int)__builtin_ctzll(reach) : (n - 1) / step;
    lo += f * step;
    n = min(step, n - f * step);
  }
  return uni(lo);
}

// Sums of two values over the threads up to each, in thread order.
__device__ __forceinline__ void block_scan(PickShared& s, u64& a, u64& b) {
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  a = wave_scan(a);
  b = wave_scan(b);
  __syncthreads();
  if (lane == kWave - 1) {
    s.part[wave] = a;
    s.part[kPickWaves + wave] = b;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPickWaves - 1; ++w) {
    const u64 x = s.part[w], y = s.part[kPickWaves + w];
    a += w < wave ? x : 0;
    b += w < wave ? y : 0;
  }
}
// Smallest key whose bin is at most b; one past `best`, the row's largest, if its bin is not either.  Bins
// fall as keys rise: every lane tries a key.
__device__ __forceinline__ uint32_t key_from(int b, uint32_t best, const RowParams& r, double base16) {
  const int lane = threadIdx.x % kWave;
  uint32_t lo = kLeastKey - 1, hi = best + 1;  // the answer is in (lo, hi]
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo - 1) / kWave + 1;
    const uint32_t c = lo + min((lane + 1) * step, hi - lo);
    double rem;
    const bool in = c == hi || min(bin_of(finite(logit_of(c)) * r.scale, base16, rem), kBins - 1) <= b;
    const int f = (int)__builtin_ctzll(__ballot(in));
    hi = min(lo + (f + 1) * step, hi);
    lo += f * step;
  }
  return uni(hi);
}

// Sorts the list, whose keys and indexes lie in the given ranges, largest first: in buckets of nearly equal
// width of the order (key, then index), then by rank in each.  False, and the list as it was, where a bucket
// holds too many: bitonic steps take 12 us for 700 tokens, 36 for 3,000; this 4 and 7.
__device__ __forceinline__ bool sort_by_bucket(PickShared& s, int n, uint32_t klo, uint32_t khi, uint32_t ilo, uint32_t ihi, int key_zeros) {
  constexpr int kPer = kList / kPickThreads;
  const int tid = threadIdx.x;
  const int index_bits = 32 - __builtin_clz((ihi - ilo) | 1u);
  // place in the order: key steps below the largest, then index
  auto place = [&](u64 w) { return ((u64)((khi >> key_zeros) - (word_key(w) >> key_zeros)) << index_bits) + (word_index(w) - ilo); };
  const u64 last = ((u64)((khi >> key_zeros) - (klo >> key_zeros)) << index_bits) + (ihi - ilo);
  int shift = 0;
  while ((last >> shift) >= (u64)kSortBuckets) ++shift;
  for (int i = tid; i < kSortBuckets; i += kPickThreads) s.bucket[i] = 0;
  __syncthreads();
  u64 word[kPer];
  uint32_t bucket[kPer], slot[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid + j * kPickThreads;
    if (i >= n) continue;
    word[j] = s.list.word[i];
    bucket[j] = (uint32_t)(place(word[j]) >> shift);
    slot[j] = atomicAdd(&s.bucket[bucket[j]], 1u);
  }
  __syncthreads();
  static_assert(kSortBuckets == 2 * kPickThreads, "two buckets per thread");
  const uint32_t c0 = s.bucket[2 * tid], c1 = s.bucket[2 * tid + 1];
  if (__syncthreads_or(max(c0, c1) > (uint32_t)kRankMost)) return false;
  u64 first = c0 + c1, none = 0;
  block_scan(s, first, none);
  s.bucket[2 * tid] = (uint32_t)first - c0 - c1;
  s.bucket[2 * tid + 1] = (uint32_t)first - c1;
  if (tid == kPickThreads - 1) s.bucket[kSortBuckets] = n;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (tid + j * kPickThreads < n) s.list.sum[s.bucket[bucket[j]] + slot[j]] = word[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (tid + j * kPickThreads >= n) continue;
    const uint32_t i0 = s.bucket[bucket[j]], i1 = s.bucket[bucket[j] + 1];
    uint32_t rank = i0;
    for (uint32_t i = i0; i < i1; ++i) rank += s.list.sum[i] > word[j];
    s.list.word[rank] = word[j];
  }
  __syncthreads();
  return true;
}

// What a pass over the row does with the tokens of bins blo..bhi, keys klo..khi and indexes ilo..ihi.
enum Act {
  kGather,    // the sorted list, with running weights (the caller knows that it fits)
  kKeyRange,  // red[0..1]: smallest and largest key
  kByKey,     // buckets of (khi - key) >> shift
  kByIndex,   // buckets of index >> shift
  kWeigh,     // the bins' weights
  kAbove,     // red[0..2]: tokens, weight and smallest order word of those with y >= y_min
};
// What the pass is for: all tokens that can be kept, or a border.
enum Step { kAll, kTopK, kTopP, kMinP, kBeforeMinP, kDraw, kDone };

template <int DT>
__global__ __launch_bounds__(kPickThreads) void sample_pick_kernel(SampleParams p) {
  constexpr int E = kVec<DT>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  PickShared& s = *(PickShared*)smem;
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const RowParams r = row_params(p, row);
  const Row<DT> x(p, row);
  const int segs = (x.vecs + kWave - 1) / kWave * kLineSegs;
  const uint32_t* seg_max = p.seg_max + (int64_t)row * p.segs;
  const ChunkHead* heads = p.heads + (int64_t)row * p.chunks;
  u64 best = 0, tokens = 0;
  double base = -INFINITY;
  for (int c = lane; c < p.chunks; c += kWave) {
    const ChunkHead h = heads[c];
    best = h.best > best ? h.best : best;
    if (h.tokens) base = fmax(base, h.base);
    tokens += h.tokens;
  }
  best = uni(wave_max_u64(best));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    base = fmax(base, __shfl_xor(base, o));
    tokens += __shfl_xor(tokens, o);
  }
  base = uni(base);
  tokens = uni(tokens);
  if (best != 0 && r.greedy) best = order_word(word_key(best), index_in(x, word_index(best), word_key(best)));
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
  const double base16 = kBinsPerLog2 * base;
  const uint32_t best_key = word_key(best);
  for (int i = tid; i < min(segs, kSegsHeld); i += kPickThreads) s.seg[i] = seg_max[i];
  if (tid < 16) s.roots[tid] = kRoots[tid];
  // ---- the row's histogram, as sums from the first bin on ----
  for (int c = tid; c < p.chunks; c += kPickThreads)  // (at most 2 kNumCu of them)
    s.down[c] = heads[c].tokens ? (int)fmin(base - heads[c].base, 64.0) : 64;
  __syncthreads();
  static_assert(kBins == kPickThreads, "a bin per thread");
  {
    u64 count = 0, weight = 0;
    const uint32_t* counts = p.counts + (int64_t)row * p.chunks * kBins;
    const u64* weights = p.weights + (int64_t)row * p.chunks * kBins;
    constexpr int kAhead = 8;
    for (int c0 = 0; c0 < p.chunks; c0 += kAhead) {
      uint32_t n[kAhead];
      u64 w[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int c = min(c0 + j, p.chunks - 1);
        const int64_t from = (int64_t)c * kBins + max(tid - kBinsPerLog2 * s.down[c], 0);
        n[j] = counts[from];
        w[j] = r.weigh ? weights[from] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int down = s.down[min(c0 + j, p.chunks - 1)];
        const bool has = c0 + j < p.chunks && tid >= kBinsPerLog2 * down && down < 64;
        count += has ? n[j] : 0;
        weight += has ? w[j] >> down : 0;
      }
    }
    block_scan(s, count, weight);
    s.count[tid] = tid == kBins - 1 ? (uint32_t)tokens : (uint32_t)count;
    s.weight[tid] = weight;
  }
  __syncthreads();
  const u64 top_k = r.top_k && (u64)r.top_k < tokens ? r.top_k : tokens;
  const float u = p.uniforms[row];
  const bool cut_p = r.top_p < 1.f, cut_m = r.min_p > 0.f;
  const double log2_min_p = cut_m ? log2(fmin((double)r.min_p, 1.0)) : -INFINITY;  // (above 1, top_k is 1)
  // min-p's border in sixteenths of log2, and its bin
  const double y_min = uni(finite(logit_of(word_key(best))) * r.scale + kBinsPerLog2 * log2_min_p);
  double rem;
  const int bin_m = uni(cut_m ? min(bin_of(y_min, base16, rem), kBins - 1) : kBins - 1);
  const int bin_k = first_reaching(s.count, kBins, top_k);
  bool weighed = r.weigh;
  constexpr int key_zeros = DT == NE_DTYPE_FP32 ? 0 : DT == NE_DTYPE_FP16 ? 13 : 16;  // low bits that a logit's type leaves the same

  // ---- passes over the row, each for one step ----
  Step step = kAll;
  Act act = kGather;
  int blo = 0, bhi = bin_k, shift = 0;  // the pass's tokens
  uint32_t klo = 1, khi = 0xFFFFFFFFu, ilo = 0, ihi = 0xFFFFFFFFu;
  bool by_count = false;  // the border: where the running count, or weight, first reaches target
  u64 target = 0, count0 = 0, weight0 = 0, left = 0;  // what lies before the pass's tokens, and how many they are
  u64 end_word = 1, end_weight = 0;  // the last kept token (1: every token), and the kept weight
  u64 border_word = 0, border_weight = 0;
  u64 reach = ~0ull;  // top-p's share of the first top_k's weight
  int all_end = kBins - 1;  // the last bin of the tokens that fit the list

  auto start_border = [&](Step what, bool count, u64 to) {
    step = what;
    by_count = count;
    target = to;
    blo = bhi = count ? first_reaching(s.count, kBins, to) : first_reaching(s.weight, kBins, to);
    count0 = uni(bhi > 0 ? (u64)s.count[bhi - 1] : 0);
    weight0 = uni(bhi > 0 ? s.weight[bhi - 1] : 0);
    left = uni((u64)s.count[bhi]) - count0;
    klo = 1;
    khi = ihi = 0xFFFFFFFFu;
    ilo = 0;
    act = left > (u64)kList ? kKeyRange : kGather;
  };
  auto start_all = [&]() {
    step = kAll;
    act = kGather;
    blo = 0;
    klo = 1;
    khi = ihi = 0xFFFFFFFFu;
    ilo = 0;
    bhi = min(bin_k, bin_m);
    if (cut_p) bhi = min(bhi, first_reaching(s.weight, kBins, reach != ~0ull ? reach : reach_at(r.top_p, uni(s.weight[bin_k]))));
    // (the exact share may pass the histogram's by some units, and with them a bin's end)
    all_end = bhi = min(bhi, all_end);
  };
  // the border of top_k is known (or there is none): top-p's, min-p's, or the draw
  auto after_top_k = [&]() {
    if (cut_p) {
      reach = reach_at(r.top_p, end_weight);
      start_border(kTopP, false, reach);
    } else {
      step = kTopP;
    }
  };
  // (a uniform of 1 takes the last kept token, which may have no weight: the row's last, unless one before it is the end)
  auto start_draw = [&]() {
    if (u >= 1.f)
      start_border(kDraw, true, tokens);
    else
      start_border(kDraw, false, draw_at(u, end_weight) + 1);
  };
  auto after_top_p = [&]() {
    // min-p can cut where a token kept so far lies in its border's bin or behind (weights do not say: one
    // below 2^-S of the largest is 0)
    const bool behind = end_word == 1 ? uni(bin_m > 0 ? (u64)s.count[bin_m - 1] : 0) < tokens
                                      : bin_of(finite(logit_of(word_key(end_word))) * r.scale, base16, rem) >= bin_m;
    if (cut_m && behind) {
      step = kMinP;
      act = kAbove;
      blo = bhi = bin_m;
      klo = 1;
      khi = ihi = 0xFFFFFFFFu;
      ilo = 0;
    } else {
      start_draw();
    }
  };
  auto first_wide = [&]() {  // a wide nucleus: each border in its own bin
    end_weight = uni(s.weight[kBins - 1]);
    if (top_k < tokens) {
      start_border(kTopK, true, top_k);
    } else {
      after_top_k();
      if (!cut_p) after_top_p();
    }
  };
  auto first = [&]() {
    start_all();
    if (uni(s.count[bhi]) > (uint32_t)kList) first_wide();
  };
  if (weighed) {
    first();
  } else if (uni(s.count[bin_k]) > (uint32_t)kList) {  // a short top-k among many nearly equal logits
    act = kWeigh;
    bhi = kBins - 2;
  }

  while (true) {
    // ---- clear ----
    __syncthreads();
    if (act == kGather) {
      if (tid == 0) s.n = 0;
    } else if (act == kByKey || act == kByIndex) {
      for (int i = tid; i < kSub; i += kPickThreads) {
        s.sub.count[i] = 0;
        s.sub.weight[i] = 0;
      }
    } else if (act == kWeigh) {
      s.weight[tid] = 0;
    }
    __syncthreads();
    // ---- the row's segments whose largest key reaches the pass's tokens, 32 at a time ----
    // (the bins as keys: an element costs two comparisons, and only those inside the rest)
    klo = max(klo, key_from(bhi, best_key, r, base16));
    khi = min(khi, blo > 0 ? key_from(blo - 1, best_key, r, base16) - 1 : best_key);
    khi -= khi == kNegativeZero;  // (as a number this end of a range would take in +0, a key above it)
    const float xlo = logit_of(klo), xhi = logit_of(khi);
    u64 acc0 = act == kKeyRange ? 0xFFFFFFFFu : 0, acc1 = 0, acc2 = ~0ull;
    for (int s0 = 0; s0 < segs && klo <= khi; s0 += kSegsHeld) {
      uint16_t* list = (uint16_t*)s.bucket;
      __syncthreads();
      if (tid == 0) s.wanted = 0;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSegsHeld / kPickThreads; ++k) {
        const int i = s0 + k * kPickThreads + tid;
        if (i >= segs || (s0 == 0 ? s.seg[i] : seg_max[i]) < klo) continue;
        list[atomicAdd(&s.wanted, 1u)] = (uint16_t)(i - s0);
      }
      __syncthreads();
      const int wanted = uni((int)s.wanted);
      constexpr int kAhead = 4;
      for (int w0 = wave * kAhead * kLineSegs; w0 < wanted; w0 += kPickWaves * kAhead * kLineSegs) {
        u32x4 raw[kAhead];
        int vec[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int at = w0 + j * kLineSegs + lane / kSegVecs;  // a segment for every 8 lanes
          vec[j] = at < wanted ? (s0 + list[at]) * kSegVecs + lane % kSegVecs : x.vecs;  // past the row
          raw[j] = x.ahead(vec[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
          if (!x.is_whole(vec[j])) raw[j] = x.vec(vec[j]);
        uint32_t inside = 0;  // one bit per element
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          float val[E];
          values<DT>(raw[j], val);
#pragma unroll
          for (int e = 0; e < E; ++e) inside |= (uint32_t)(val[e] >= xlo && val[e] <= xhi) << (j * E + e);
        }
        while (inside) {
          const int bit = __builtin_ctz(inside);
          inside &= inside - 1;
          int of = vec[0];
          uint32_t dword = raw[0][0];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            of = bit >= j * E ? vec[j] : of;
#pragma unroll
            for (int d = 0; d < 4; ++d) dword = bit >= j * E + d * E / 4 ? raw[j][d] : dword;
          }
          const int t = of * E + bit % E - x.skew;
          if ((uint32_t)t < ilo || (uint32_t)t > ihi) continue;
          const float v = element<DT>(dword, bit % (E / 4));
          const uint32_t k = key_of(v);
          if (act == kGather) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < (uint32_t)kList) s.list.word[at] = order_word(k, t);
            continue;
          }
          const double y16 = finite(v) * r.scale;
          const int b = bin_of(y16, base16, rem);
          const u64 w = b < kBins ? weight_int(weight_of(b, rem, p.weight_exp, s.roots)) : 0;
          if (act == kKeyRange) {
            acc0 = k < acc0 ? k : acc0;
            acc1 = k > acc1 ? k : acc1;
          } else if (act == kWeigh) {
            atomicAdd(&s.weight[b], w);
          } else if (act == kAbove) {
            if (y16 >= y_min) {
              const u64 o = order_word(k, t);
              ++acc0;
              acc1 += w;
              acc2 = o < acc2 ? o : acc2;
            }
          } else {
            const uint32_t c = act == kByKey ? (khi - k) >> shift : (uint32_t)t >> shift;
            atomicAdd(&s.sub.count[c], 1u);
            atomicAdd(&s.sub.weight[c], w);
          }
        }
      }
    }
    __syncthreads();
    // ---- what the pass found ----
    if (act == kWeigh) {
      u64 w = s.weight[tid], none = 0;
      block_scan(s, w, none);
      s.weight[tid] = w;
      __syncthreads();
      weighed = true;
      first();
      continue;
    }
    if (act == kKeyRange || act == kAbove) {
      if (act == kKeyRange) {
        acc0 = ~wave_max_u64(~acc0);
        acc1 = wave_max_u64(acc1);
      } else {
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
          acc0 += __shfl_xor(acc0, o);
          acc1 += __shfl_xor(acc1, o);
        }
        acc2 = ~wave_max_u64(~acc2);
      }
      u64* all = s.list.sum;  // [3][waves], the list is not in use
      if (lane == 0) {
        all[wave] = acc0;
        all[kPickWaves + wave] = acc1;
        all[2 * kPickWaves + wave] = acc2;
      }
      __syncthreads();
      for (int w = 0; w < kPickWaves; ++w) {
        if (w == wave) continue;
        const u64 a = all[w], b = all[kPickWaves + w], c = all[2 * kPickWaves + w];
        if (act == kKeyRange) {
          acc0 = a < acc0 ? a : acc0;
          acc1 = b > acc1 ? b : acc1;
        } else {
          acc0 += a;
          acc1 += b;
          acc2 = c < acc2 ? c : acc2;
        }
      }
    }
    if (act == kAbove) {
      const u64 before = uni(bin_m > 0 ? (u64)s.count[bin_m - 1] : 0);
      acc0 = uni(acc0);
      acc1 = uni(acc1);
      acc2 = uni(acc2);
      if (acc0 > 0) {
        if (acc2 > end_word) {
          end_word = acc2;
          end_weight = uni(bin_m > 0 ? s.weight[bin_m - 1] : 0) + acc1;
        }
        start_draw();
      } else if (before > 0) {  // no token of its bin: the last kept one is the last before the bin
        start_border(kBeforeMinP, true, before);
      } else {
        start_draw();
      }
      continue;
    }
    if (act == kKeyRange) {
      klo = uni((uint32_t)acc0);
      khi = uni((uint32_t)acc1);
    } else if (act == kByKey || act == kByIndex) {
      static_assert(kSub == 2 * kPickThreads, "two buckets per thread");
      const u64 a = s.sub.count[2 * tid], b = s.sub.weight[2 * tid];
      u64 sa = a + s.sub.count[2 * tid + 1], sb = b + s.sub.weight[2 * tid + 1];
      const u64 ta = sa, tb = sb;
      block_scan(s, sa, sb);
      s.sub.count[2 * tid] = (uint32_t)(sa - ta + a);
      s.sub.weight[2 * tid] = sb - tb + b;
      s.sub.count[2 * tid + 1] = (uint32_t)sa;
      s.sub.weight[2 * tid + 1] = sb;
      __syncthreads();
      const u64 most = uni(s.sub.weight[kSub - 1]);
      // (the histogram's sums may differ from these tokens' in the last place: a weight past them is their end)
      const int c = by_count || act == kByIndex ? first_reaching(s.sub.count, kSub, target - count0)
                                                : first_reaching(s.sub.weight, kSub, min(target - weight0, most));
      const u64 had = uni(c > 0 ? (u64)s.sub.count[c - 1] : 0);
      left = uni((u64)s.sub.count[c]) - had;
      count0 += had;
      weight0 += uni(c > 0 ? s.sub.weight[c - 1] : 0);
      if (act == kByKey) {
        const uint32_t top = khi - ((uint32_t)c << shift);
        klo = max(klo, top - ((1u << shift) - 1u));
        khi = top;
      } else {
        ilo = (uint32_t)c << shift;
        ihi = ilo + (1u << shift) - 1u;
      }
    }
    if (act != kGather) {  // narrower, until the tokens fit the list
      if (left <= (u64)kList) {
        act = kGather;
      } else if (klo < khi) {
        act = kByKey;
        shift = 0;
        while (((khi - klo) >> shift) >= (uint32_t)kSub) ++shift;
      } else {  // one logit: from here on a rank decides, and the index finds it
        if (!by_count) {
          const u64 w = uni(weight_of_key(klo, r, base16, p.weight_exp, s.roots));
          u64 rank = w ? (target - weight0 + w - 1) / w : 1;
          rank = min(max(rank, (u64)1), left);
          by_count = true;
          target = count0 + rank;
        }
        act = kByIndex;
        shift = 0;
        while (((uint32_t)(p.vocab - 1) >> shift) >= (uint32_t)kSub) ++shift;
      }
      continue;
    }
    // ---- sort the list, largest first ----
    const int n = uni(min((int)s.n, kList));
    if (n <= 256) {  // each token counts those before it
      const u64 mine = tid < n ? s.list.word[tid] : 0;
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += s.list.word[i] > mine;
      __syncthreads();
      if (tid < n) s.list.word[rank] = mine;
      __syncthreads();
    } else if (sort_by_bucket(s, n, klo, khi, ilo, min(ihi, (uint32_t)p.vocab - 1), key_zeros)) {
    } else {
      int size = 512;
      while (size < n) size <<= 1;
      for (int i = n + tid; i < size; i += kPickThreads) s.list.word[i] = 0;
      __syncthreads();
      for (int k = 2; k <= size; k <<= 1) {  // bitonic
        for (int j = k >> 1; j > 0; j >>= 1) {
          for (int t = tid; t < size / 2; t += kPickThreads) {
            const int a = 2 * t - (t & (j - 1));
            const u64 c = s.list.word[a], d = s.list.word[a + j];
            if (((a & k) == 0) ? c < d : c > d) {
              s.list.word[a] = d;
              s.list.word[a + j] = c;
            }
          }
          __syncthreads();
        }
      }
    }
    {  // running weights: each thread a run of consecutive entries
      const int per = (n + kPickThreads - 1) / kPickThreads;
      const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
      u64 mine = 0, none = 0;
      for (int i = i0; i < i1; ++i) {
        mine += weight_of_key(word_key(s.list.word[i]), r, base16, p.weight_exp, s.roots);
        s.list.sum[i] = mine;
      }
      u64 incl = mine;
      block_scan(s, incl, none);
      for (int i = i0; i < i1; ++i) s.list.sum[i] += incl - mine;
      __syncthreads();
    }
    if (step == kAll) {
      // every token that can be kept is in the list; top-p's share is of the first top_k's weight: the
      // list's, or, where the list ends before them, the histogram's
      const int nk = (int)min(top_k, (u64)n);
      if (cut_p && reach == ~0ull) {
        if ((u64)nk == top_k) {
          reach = reach_at(r.top_p, uni(s.list.sum[nk - 1]));
        } else if (top_k == tokens) {
          reach = reach_at(r.top_p, uni(s.weight[kBins - 1]));
        } else {
          start_border(kTopK, true, top_k);
          end_weight = ~0ull;  // and back here, with reach
          continue;
        }
      }
      u64 kept_p = 0, kept_m = 0;
      for (int i = tid; i < nk; i += kPickThreads) {
        kept_p += i == 0 || s.list.sum[i - 1] < reach;
        kept_m += finite(logit_of(word_key(s.list.word[i]))) * r.scale >= y_min;
      }
      block_scan(s, kept_p, kept_m);
      if (tid == kPickThreads - 1) {
        s.red[0] = kept_p;
        s.red[1] = kept_m;
      }
      __syncthreads();
      const int kept = uni(max(1, min((int)min(s.red[0], s.red[1]), nk)));
      const u64 sum = uni(s.list.sum[kept - 1]);
      const int at = u >= 1.f ? kept - 1 : first_reaching(s.list.sum, kept, draw_at(u, sum) + 1);
      end_word = uni(s.list.word[kept - 1]);
      end_weight = sum;
      border_word = uni(s.list.word[at]);
      break;
    }
    // ---- a border ----
    {
      const int i = by_count ? (int)min(target - count0, (u64)n) - 1 : first_reaching(s.list.sum, n, target - weight0);
      border_word = uni(s.list.word[max(i, 0)]);
      border_weight = weight0 + uni(s.list.sum[max(i, 0)]);
    }
    if (step == kTopK && end_weight == ~0ull) {
      reach = reach_at(r.top_p, border_weight);
      end_weight = 0;
      start_all();
      continue;
    }
    if (step == kDraw) break;
    if (border_word > end_word) {
      end_word = border_word;
      end_weight = border_weight;
    }
    if (step == kTopK) {
      after_top_k();
      if (!cut_p) after_top_p();
    } else if (step == kTopP) {
      after_top_p();
    } else {
      start_draw();
    }
  }
  if (tid == 0) {
    // sums of a bin's tokens and of the histogram may differ in the last place
    p.tokens[row] = (int32_t)word_index(border_word > end_word || end_word == 1 ? border_word : end_word);
    out.last = end_word;
    out.sum = ldexp((double)end_weight, -p.weight_exp);
    p.results[row] = out;
  }
}

// ---- probs ----
constexpr int kProbsThreads = 256;
constexpr int kProbsPer = 2;  // vectors per thread
constexpr int kFarBins = 16 * 160;  // below 2^-160 a probability is 0 in fp32

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
  const double inv = 1.0 / r.sum, base16 = kBinsPerLog2 * r.base;
  float* to = p.probs + (int64_t)row * p.ld_probs;
  u32x4 raw[kProbsPer];
#pragma unroll
  for (int j = 0; j < kProbsPer; ++j) raw[j] = x.ahead(v0 + j * kProbsThreads);
#pragma unroll
  for (int j = 0; j < kProbsPer; ++j) {
    const int v = v0 + j * kProbsThreads;
    if (v >= x.vecs) continue;
    if (!x.is_whole(v)) raw[j] = x.vec(v);
    float val[E], out[E];
    values<DT>(raw[j], val);
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
        const int b = bin_of(finite(val[e]) * r.scale, base16, rem);
        out[e] = b < kFarBins ? (float)(weight_of(b, rem, 0, s_roots) * inv) : 0.f;
      }
    }
    if (t0 >= 0 && t0 + E <= x.vocab && ((uintptr_t)(to + t0) & 15) == 0) {
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

// Chunks of a row.  fp32: enough work-groups to fill the chip twice, at least one iteration of the scan each;
// 16 bits: a work-group per CU, of three lines per wave at least, as each adds a histogram to merge (one to
// eight rows 26 to 27 us, 27 to 28 with one line).
int row_chunks(int rows, int lines, int dtype) {
  rows = rows < 1 ? 1 : rows;
  const int want = ceil_div(dtype == NE_DTYPE_FP32 ? 2 * kNumCu : kNumCu, rows);
  const int most = ceil_div(lines, dtype == NE_DTYPE_FP32 ? kScanWaves * kScanLines : kCountLeast);
  const int n = want < most ? want : most, least = ceil_div(lines, kCountMost);
  return dtype == NE_DTYPE_FP32 || n > least ? n : least;
}

struct Layout {
  int chunks, segs;
  size_t heads, counts, weights, seg_max, results, bytes;
};
Layout layout_of(int rows, int vocab, int dtype) {
  Layout l;
  const int e = elements_per_vec(dtype);
  rows = rows < kRowBatch ? rows : kRowBatch;
  const int lines = ceil_div(vocab + e - 1, e * kWave);  // a row off the 16-byte grid may touch one vector more
  l.segs = lines * kLineSegs;
  l.chunks = row_chunks(rows, lines, dtype);
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
  if constexpr (DT == NE_DTYPE_FP32) {
    hipLaunchKernelGGL(sample_scan_kernel, dim3(p.chunks, p.rows), dim3(kScanThreads), 0, s, p);
  } else {
    static const hipError_t attr = hipFuncSetAttribute((const void*)sample_count_kernel<DT>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(CountShared<DT>));
    if (attr != hipSuccess) {
      set_error("sample_count: cannot reserve %d bytes of LDS: %s", (int)sizeof(CountShared<DT>), hipGetErrorString(attr));
      return NE_ELAUNCH;
    }
    hipLaunchKernelGGL(sample_count_kernel<DT>, dim3(p.chunks, p.rows), dim3(kCountThreads), sizeof(CountShared<DT>), s, p);
  }
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
