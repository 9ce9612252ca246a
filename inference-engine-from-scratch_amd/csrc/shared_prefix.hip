// Attention of a batch whose sequences share prefixes: the keys of a shared prefix are
// read once for all its sequences' queries, the rest per sequence.
//
// Mathematics.  A query row's keys are cut into parts; part a gives its largest score m_a
// (or a reference below which nothing is lost), l_a = sum 2^(s - m_a) and
// O_a = sum 2^(s - m_a) v, and the row is sum_a 2^(m_a - M) O_a / sum_a 2^(m_a - M) l_a.
// Which rows compute a part together does not matter, so a prefix's parts serve every
// row of its group (a matrix product of all their queries with the shared keys) and the
// rest of each sequence has parts of its own.
//
// Three kernels.
//   plan   one work-group, once per step for all layers: the groups' common lengths from
//          the sequences' present ones (a member may be idle, a group may shrink to one),
//          the tokens of each group in order, and the work items.
//   parts  an item is one of
//            a tile of 64, 128 or 256 rows of a group (tokens x heads of one KV head) over a
//            range of the prefix, or of one sequence with more than 32 rows per KV head over
//            a range of its own keys: 128 keys at a time staged in LDS as MFMA operands,
//            eight waves of 32 rows (qt_* in attention_tile.hpp), key groups where rows are
//            few;
//            a light item: a range of the own keys of one sequence with at most 32 rows per
//            KV head: one wave per KV head, K and V straight from memory to registers, the
//            rows as the second operand of S^T = K Q^T, whose result is the second operand of
//            O^T = V^T P^T.
//          Items are cut so that the longest is about the batch's work over the chip.
//   merge  16 threads per row, or 64.
// What bounds it: reading the keys once (long prefixes and contexts), else the chain of
// round trips of the three kernels; the partial sums (520 bytes a row and part) stay in the
// memory-side cache.
//
// int8 pools: codes become fp16 exactly, the key scale multiplies the score, the value
// scale the probability.  Probabilities enter the second product with 16 bits (11 significant
// ones for int8 pools, 8 for bf16 pools, as the values themselves have): each is off by at
// most half a step, and those errors average over the keys.  Value scales are taken relative
// to a power of two that follows the largest met so far, so that small scales keep their bits in fp16.
// A key that a row does not see never reaches it, whatever its value holds: values of partly
// hidden keys that are not finite enter the products as 0, and the merge adds them to the rows
// that see them.
#include <string.h>

#include <type_traits>

#include "attention_tile.hpp"

namespace ne {

namespace {

constexpr int kSpThreads = kQtThreads;
constexpr int kSpWaves = kQtWaves;
constexpr int kSpMaxSeqs = 1024;
constexpr int kLightRows = 32;       // rows per KV head of a light item
constexpr int kLightMinTiles = 4;    // least 16-key tiles per wave of a split sequence
// The plan's costs, in the time of 16 keys of a light item that waits for nothing else (0.6 us).
// A stage of a tile of up to 128 rows waits for its keys as much as it computes (2.9 us), one of 256 computes.
constexpr int kStageCost = 5, kBigStageCost = 9;
constexpr int kItemCost = 13;  // an item before its first and after its last keys: 6.5 us (light) to 10 (tile)
// With this many tiles of 16 keys of eight heads (and as large stages of a head) per CU, 50 MB of an int8
// pool, they come at the memory's rate.  64 rows on 16,384 keys (bf16) 124 us with the cost of 3, 132 with 2,
// 161 with 1; nine prefixes of 2,048 keys that leave little (int8) 46 with 4 tiles, 39 with 6.
constexpr int kStreamTiles = 6, kStreamCost = 3;
__host__ __device__ constexpr int stage_cost(int tile_rows) { return tile_rows <= 128 ? kStageCost : kBigStageCost; }
// Sharing has to save this much per CU, and this part of the light work: a tile item takes longer than a light
// one, the more so beside others that stream, and its partial sums go through memory.  32 sequences of 9 rows
// whose own keys are ten times the shared ones: 367 us shared, 326 not.
constexpr int kShareGain = 3, kShareOf = 8;
// Tiles of 256 rows take a tenth less per row; worth it with this much tile work per CU, as half tiles
// spread it better.
constexpr int kBigWork = 60;
constexpr int kSpSeqInts = 10;
constexpr float kSpLazy = 256.f;     // probabilities' sum per lane and step before the reference moves

// A work-group's item, as the plan writes it.
enum : int32_t { kGroupTile = 0, kOwnTile = 1, kLight = 2 };
struct SpItem {
  int32_t kind;
  int32_t seq;         // whose block table is read
  int32_t head;        // KV head (light: first of the work-group's)
  int32_t rows_total;  // query rows per KV head of the group, or sequence
  int32_t row0;        // tile: its first row, and the rows of a tile
  int32_t tile_rows;
  int32_t token;       // group tile: its first token in `tokens`; else the sequence's first row of q
  int32_t first_seen;  // keys that query 0 sees (a later one sees one more each); group tile: all
  int32_t k0, k1;      // keys
  int32_t part_row;    // first partial row of KV head 0 (light: and of part 0)
  int32_t part0, parts, tiles;  // light: its first wave's part of `parts` over `tiles` tiles from k0 on
  int32_t pad[2];
};
static_assert(sizeof(SpItem) == 64, "");

// What bits of the error word mean.
enum : uint32_t { kErrContext = 1, kErrRows = 2, kErrGroups = 4, kErrBlock = 8 };

struct SpParams {
  const uint16_t* q;
  int64_t q_tok_stride, q_head_stride;
  const void* k_cache;
  const void* v_cache;
  const void* k_scale;
  const void* v_scale;
  const int32_t* block_tables;
  int32_t bt_stride, block_size, num_blocks;
  const int32_t* ctx_len;
  const int32_t* q_start;
  const int32_t* q_len;
  const int32_t* group_seqs;
  const int32_t* group_start;
  const int32_t* prefix_len;
  int32_t num_seqs, num_groups, num_rows;  // num_rows: query tokens of q and out
  int32_t num_kv_heads, group;             // group: query heads per KV head
  int32_t max_q, max_ctx;
  float qk_scale;  // softmax_scale * log2(e)
  uint16_t* out;
  int64_t o_tok_stride, o_head_stride;
  // workspace
  uint32_t* head;      // [0] error word, [1] items, [2] of them of shared prefixes
  int32_t* tokens;     // row of q of every group's tokens, group after group
  SpItem* items;       // [max_items]: tiles, then light items
  int32_t* seqs;       // [num_seqs][kSpSeqInts]
  float* part_o;       // [parts' rows][128]
  float* part_ml;      // [parts' rows][2]
  int32_t max_items;
  int32_t light_heads, light_keys;  // a light work-group's KV heads, and its waves per KV head
  int32_t head_blocks;              // work-groups per light item
  int64_t part_rows;
};

__host__ __device__ inline int cdiv(int a, int b) { return (a + b - 1) / b; }
// Rows of the tiles that `rows` rows are cut into: 64, 128, or (big, if that fills them) 256.
__host__ __device__ inline int tile_rows_of(int rows, bool big) {
  return rows <= 64 ? 64 : !big || cdiv(rows, 256) * 256 * 8 > cdiv(rows, 128) * 128 * 9 ? 128 : 256;
}

// ---- plan ----
constexpr int kPlanMaxThreads = kSpMaxSeqs;

// Sums of K values over the threads before each, and over all, in two barriers.
template <int K>
__device__ __forceinline__ void plan_scan(const int (&v)[K], int (*s_part)[kPlanMaxThreads / kWave], int (&before)[K], int (&total)[K]) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  int incl[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {  // within rows of 16 lanes, then over rows
    int x = v[k];
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    incl[k] = x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  }
  __syncthreads();
  if (lane == kWave - 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) s_part[k][wave] = incl[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    before[k] = incl[k] - v[k];
    total[k] = 0;
    for (int w = 0; w < waves; ++w) {
      const int x = s_part[k][w];
      before[k] += w < wave ? x : 0;
      total[k] += x;
    }
  }
}
// Largest i in [0, n) with first[i] <= x (first[0] <= x).
__device__ __forceinline__ int last_from(const int* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first[mid] <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ int ceil_share(int64_t work, int workers) { return (int)((work + workers - 1) / workers); }

// One work-group of a thread per sequence; thread e serves entry e of the groups' list, group e and
// sequence e.  (Counts fit 32 bits: the host bounds the workspace's rows.)
__global__ __launch_bounds__(kPlanMaxThreads) void shared_prefix_plan_kernel(SpParams p, int max_prefix) {
  __shared__ int s_part[5][kPlanMaxThreads / kWave];
  __shared__ int s_start[kSpMaxSeqs + 1];   // groups' first entries
  __shared__ int s_least[kSpMaxSeqs];       // per group: fewest keys before a member's queries
  __shared__ int s_leader[kSpMaxSeqs];      // first active entry
  __shared__ int s_members[kSpMaxSeqs];
  __shared__ int s_prefix[kSpMaxSeqs];      // keys shared (0: none)
  __shared__ int s_token0[kSpMaxSeqs + 1];  // per entry: its first token
  __shared__ int s_row[kSpMaxSeqs];         // per entry: its first row of q
  __shared__ int s_owner[kSpMaxSeqs];       // per sequence: its first entry
  __shared__ int s_alone[kSpMaxSeqs];       // per group: units of its prefix read by every member
  __shared__ int s_parts[kSpMaxSeqs];       // per group
  __shared__ int s_item0[kSpMaxSeqs];       // per group: its first tile item
  __shared__ int s_row0[kSpMaxSeqs];        // per group: its first partial row
  const int e = threadIdx.x, threads = blockDim.x;
  const int n = p.num_seqs, G = p.num_groups;
  uint32_t error = 0;
  int seq = e < n ? p.group_seqs[e] : -1;
  const int stated = e < G ? p.prefix_len[e] : 0;
  if (e < G) {
    s_start[e] = p.group_start[e];
    s_least[e] = 0x7FFFFFFF;
    s_leader[e] = 0x7FFFFFFF;
    s_members[e] = 0;
  }
  if (e == 0) {
    s_start[G] = p.group_start[G];
    p.head[0] = 0;
  }
  if (e < n) {
    s_owner[e] = 0x7FFFFFFF;
    p.seqs[(int64_t)e * kSpSeqInts] = 0;  // a sequence that no entry names has no rows
  }
  // ---- entry e of the groups' list ----
  int ctx = 0, ql = 0, qs = 0;
  if (e < n) {
    if (seq < 0 || seq >= n) {
      error |= kErrGroups;
      seq = -1;
    } else {
      ctx = p.ctx_len[seq];
      ql = p.q_len[seq];
      qs = p.q_start[seq];
      if (ql > p.max_q || (ql > 0 && (qs < 0 || qs > p.num_rows - ql))) {
        error |= kErrRows;
        ql = 0;
      }
      if (ctx > p.max_ctx) error |= kErrContext;
      if (ctx <= 0) ql = 0;
      ql = max(ql, 0);
    }
  }
  __syncthreads();
  if (seq >= 0) atomicMin(&s_owner[seq], e);
  __syncthreads();
  if (seq >= 0 && s_owner[seq] != e) {  // named twice: the first entry counts
    error |= kErrGroups;
    seq = -1;
    ql = 0;
  }
  if (e == 0 && (s_start[0] != 0 || s_start[G] != n)) error |= kErrGroups;
  if (e < G && s_start[e] > s_start[e + 1]) error |= kErrGroups;
  // the sequence's group: a list that does not start at 0, or ends early, leaves singles
  int g = -1;
  if (e < n && G > 0 && s_start[0] <= e && e < s_start[G]) {
    g = last_from(s_start, G, e);
    if (s_start[g] > e || e >= s_start[g + 1]) g = -1;  // not in order
  }
  if (e < n && g < 0) error |= kErrGroups;
  if (ql > 0 && g >= 0) {
    atomicMin(&s_least[g], max(ctx - ql, 0));
    atomicMin(&s_leader[g], e);
    atomicAdd(&s_members[g], 1);
  }
  const int table_keys = (int)min((int64_t)p.bt_stride * p.block_size, (int64_t)0x7FFFFFFF);
  const int rows_s = ql * p.group;
  const bool light = rows_s <= kLightRows;
  const int kend = min(min(ctx, p.max_ctx), table_keys);
  // tokens, and the light work if no prefix were shared (of up to 2^27 / 1,024 keys a sequence)
  int before[2], total[2];
  plan_scan<2>({ql, ql > 0 && light ? min(cdiv(max(kend, 0), kTileKeys) * p.head_blocks / p.light_keys, 1 << 20) : 0}, s_part, before, total);
  const int t0 = before[0], tokens = total[0];
  auto stream_of = [&](float tiles) { return tiles >= (float)(kStreamTiles * kNumCu) ? kStreamCost : 1; };
  const int stream_alone = stream_of((float)total[1]);
  if (e < n) {
    s_token0[e] = t0;
    s_row[e] = qs;
  }
  if (e == 0) s_token0[n] = tokens;
  __syncthreads();
  auto first_token = [&](int entry) { return s_token0[min(max(entry, 0), n)]; };
  // ---- group e ----
  int rows = 0, stages = 0, prefix = 0;
  if (e < G && s_members[e] > 1) {
    prefix = min(min(stated, s_least[e]), min(max_prefix, p.max_ctx));
    prefix = max(min(prefix, table_keys), 0) & ~(kTileKeys - 1);
    if (prefix > 0) {
      rows = (first_token(s_start[e + 1]) - first_token(s_start[e])) * p.group;
      stages = cdiv(prefix, kQtKeys);
    }
  }
  if (e < G) {
    s_prefix[e] = prefix;
    s_alone[e] = 0;
  }
  __syncthreads();
  // ---- what the prefixes would cost read by every member ----
  if (ql > 0 && g >= 0 && s_prefix[g] > 0) {
    const int64_t units = light ? (int64_t)(s_prefix[g] / kTileKeys) * p.head_blocks * stream_alone / p.light_keys
                                : (int64_t)cdiv(rows_s, 128) * cdiv(s_prefix[g], kQtKeys) * kStageCost * p.num_kv_heads;
    atomicAdd(&s_alone[g], (int)min(units, (int64_t)1 << 20));
  }
  __syncthreads();
  const int64_t shared = (int64_t)cdiv(rows, 128) * stages * kStageCost * p.num_kv_heads;
  const bool gains = e < G && prefix > 0 && s_alone[e] > shared;
  int skip[3], sum[3];
  // (capped so that the sums stay in 32 bits)
  plan_scan<3>({gains ? (int)min(s_alone[e] - shared, (int64_t)1 << 20) : 0, gains ? min(cdiv(rows, 128) * stages, 1 << 20) : 0,
                light ? 0 : min(cdiv(rows_s, 128) * cdiv(max(kend, 0), kQtKeys), 1 << 20)},
               s_part, skip, sum);
  const bool big = ((int64_t)sum[1] + sum[2]) * p.num_kv_heads * kStageCost >= (int64_t)kBigWork * kNumCu;
  if (!gains || sum[0] < max(kShareGain * kNumCu, total[1] / kShareOf * stream_alone)) prefix = rows = stages = 0;
  const int tile_rows = tile_rows_of(rows, big), tile_count = cdiv(rows, tile_rows);
  if (e < G) s_prefix[e] = prefix;
  __syncthreads();
  // ---- entry e: its own keys ----
  const int from = g >= 0 ? s_prefix[g] : 0;
  const int own = ql > 0 ? max(kend - from, 0) : 0;
  const int tile_rows_s = tile_rows_of(rows_s, big);
  const int tiles16 = light ? cdiv(own, kTileKeys) : 0;
  const int heavy_tiles = light || own == 0 ? 0 : cdiv(rows_s, tile_rows_s);
  const int heavy_stages = light ? 0 : cdiv(own, kQtKeys);
  // ---- the batch's work, and a work-group's share of it ----
  // Each item, one work-group and one per CU at a time, gets keys worth x, so that all take about as long
  // as the chip takes for the batch: with work W and B uncut items, W / x further ones,
  //   kNumCu (x + F) = W + F (B + W / x), F = kItemCost.
  // x >= W / kNumCu for any B, so there are kNumCu further items at most.
  float x;
  int stream;
  {
    const int64_t mine = ((int64_t)tile_count * stages * stage_cost(tile_rows) + (int64_t)heavy_tiles * heavy_stages * stage_cost(tile_rows_s)) * p.num_kv_heads;
    int before[5], total[5];  // (of this block) tile work (1,024 of 48 bits), light work, and uncut items
    plan_scan<5>({(int)(mine & 0xFFFF), (int)((mine >> 16) & 0xFFFF), (int)(mine >> 32), tiles16,
                  min((tile_count + heavy_tiles) * p.num_kv_heads + (tiles16 > 0 ? p.head_blocks : 0), 1 << 20)},
                 s_part, before, total);
    const float tile_work = (float)total[0] + 65536.f * (float)total[1] + 4294967296.f * (float)total[2];
    const float light_work = (float)total[3] * (float)p.head_blocks / (float)p.light_keys;
    stream = stream_of(light_work + tile_work / (float)kStageCost);
    const float W = tile_work + light_work * (float)stream, B = (float)total[4];
    constexpr float F = kItemCost, C = kNumCu;
    const float b = C * F - W - F * B;
    x = fmaxf((sqrtf(b * b + 4.f * C * F * W) - b) / (2.f * C), W / C);
  }
  // n / each rounded, 1 at least and n at most
  auto parts_of = [](int n, float each) { return n > 0 ? min(max((int)((float)n / each + 0.5f), 1), n) : 0; };
  auto stages_each = [&](int tr) { return fmaxf(x / (float)stage_cost(tr), 1.f); };
  const int parts = parts_of(stages, stages_each(tile_rows));
  const int parts_s = light ? parts_of(tiles16, fmaxf(x / (float)stream, (float)kLightMinTiles)) : parts_of(heavy_stages, stages_each(tile_rows_s));
  const int light_items = light ? cdiv(parts_s, p.light_keys) : 0;
  // tile items of groups, their partial rows; light items, tile items and partial rows of sequences
  int at[5], all[5];
  plan_scan<5>({tile_count * parts, rows * parts * p.num_kv_heads, light_items, heavy_tiles * parts_s, rows_s * parts_s * p.num_kv_heads},
               s_part, at, all);
  if (e < G) {
    s_parts[e] = parts;
    s_item0[e] = at[0];
    s_row0[e] = at[1];
  }
  __syncthreads();
  const int items = all[0];
  const int srow0 = all[1] + at[4];
  const int tile_wgs = (items + all[3]) * p.num_kv_heads, light_wgs = all[2] * p.head_blocks;
  // (the workspace's bounds hold for any lengths and groups in order; a list out of order may exceed them)
  const bool fits = tile_wgs + light_wgs <= p.max_items && (int64_t)all[1] + all[4] <= p.part_rows;
  if (!fits) error |= kErrGroups;
  if (seq >= 0) {
    int32_t* d = p.seqs + (int64_t)seq * kSpSeqInts;
    const int group_token0 = g >= 0 ? first_token(s_start[g]) : 0;
    d[0] = fits ? ql : 0;
    d[1] = qs;
    d[2] = from > 0 ? s_parts[g] : 0;  // parts of the shared prefix
    d[3] = parts_s;                    // parts of its own keys
    d[4] = g >= 0 ? s_row0[g] + (t0 - group_token0) * p.group : 0;
    d[5] = g >= 0 ? (first_token(s_start[g + 1]) - group_token0) * p.group : 0;
    d[6] = srow0;
    d[7] = rows_s;
    d[8] = ctx;
    d[9] = 0;  // set where a partly hidden key's value is not finite
  }
  if (e == 0) {
    p.head[1] = fits ? (uint32_t)(tile_wgs + light_wgs) : 0;
    p.head[2] = fits ? (uint32_t)(items * p.num_kv_heads) : 0;  // of them, of shared prefixes
  }
  if (error) atomicOr(p.head, error);
  if (!fits) return;
  // ---- the groups' tokens, and the items ----
  for (int i = e; i < tokens; i += threads) {
    const int k = last_from(s_token0, n, i);  // (of entries with the same first token, the last holds it)
    p.tokens[i] = s_row[k] + i - s_token0[k];
  }
  for (int x = e; x < items * p.num_kv_heads; x += threads) {
    const int i = x / p.num_kv_heads;
    const int k = last_from(s_item0, G, i);
    const int first = s_start[k];
    const int rows_g = (first_token(s_start[k + 1]) - first_token(first)) * p.group;
    const int tr = tile_rows_of(rows_g, big), count = cdiv(rows_g, tr);
    const int tile = (i - s_item0[k]) % count, part = (i - s_item0[k]) / count;
    const int st = cdiv(s_prefix[k], kQtKeys);
    SpItem d = {};
    d.kind = kGroupTile;
    d.seq = p.group_seqs[s_leader[k]];
    d.head = x % p.num_kv_heads;
    d.rows_total = rows_g;
    d.row0 = tile * tr;
    d.tile_rows = tr;
    d.token = first_token(first);
    d.first_seen = 0x7FFFFFFF;
    d.k0 = (int)((int64_t)st * part / s_parts[k]) * kQtKeys;
    d.k1 = min((int)((int64_t)st * (part + 1) / s_parts[k]) * kQtKeys, s_prefix[k]);
    d.part_row = s_row0[k] + part * p.num_kv_heads * rows_g;
    p.items[x] = d;
  }
  // entry e's own items (few each)
  if (seq >= 0 && parts_s > 0) {
    SpItem d = {};
    d.seq = seq;
    d.rows_total = rows_s;
    d.token = qs;
    d.first_seen = ctx - ql + 1;
    for (int x = 0; x < heavy_tiles * parts_s * p.num_kv_heads; ++x) {
      const int i = x / p.num_kv_heads, tile = i % heavy_tiles, part = i / heavy_tiles;
      d.kind = kOwnTile;
      d.head = x % p.num_kv_heads;
      d.row0 = tile * tile_rows_s;
      d.tile_rows = tile_rows_s;
      d.k0 = from + (int)((int64_t)heavy_stages * part / parts_s) * kQtKeys;
      d.k1 = min(from + (int)((int64_t)heavy_stages * (part + 1) / parts_s) * kQtKeys, kend);
      d.part_row = srow0 + part * p.num_kv_heads * rows_s;
      p.items[(items + at[3]) * p.num_kv_heads + x] = d;
    }
    for (int x = 0; x < light_items * p.head_blocks; ++x) {
      d.kind = kLight;
      d.head = x % p.head_blocks * p.light_heads;
      d.k0 = from;
      d.k1 = kend;
      d.part_row = srow0;
      d.part0 = x / p.head_blocks * p.light_keys;
      d.parts = parts_s;
      d.tiles = tiles16;
      p.items[tile_wgs + at[2] * p.head_blocks + x] = d;
    }
  }
}

// ---- a row's state ----
template <bool INT8>
struct SpState {
  QFrag<INT8> q[kQtMT];
  float m[kQtMT], l[kQtMT];
  floatx4 o[kQtMT][8];
};

template <bool INT8>
__device__ __forceinline__ floatx4 sp_mfma(u32x4 a, const std::conditional_t<INT8, f16x8, bf16x8>& b, floatx4 c) {
  if constexpr (INT8)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), b, c, 0, 0, 0);
}

// 16 bytes of a query row as a B operand (bf16 -> fp16 is exact for |q| in [2^-14, 65504), and
// rounds smaller ones to 2^-25).
template <bool INT8>
__device__ __forceinline__ auto sp_q_operand(u32x4 raw) {
  if constexpr (INT8) {
    u32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = pack_f16x2(bf16_to_f32((uint16_t)(raw[i] & 0xFFFFu)), bf16_to_f32((uint16_t)(raw[i] >> 16)));
    return __builtin_bit_cast(f16x8, h);
  } else {
    return __builtin_bit_cast(bf16x8, raw);
  }
}

// Probabilities of a 32-key step for MT row tiles: s[mt][t][i] is the score of key 16 t + 4 g + i.
// kf / vf: the keys' score factors and value factors (int8).  hidden(mt, e): key of slot e = 4 t + i
// is not seen.  down: what the outputs so far shrink by (1: nothing changed).  Returns the second
// product's operands in pb.
template <bool INT8, int MT, typename Hidden>
__device__ __forceinline__ void sp_softmax(const floatx4 (&s)[MT][2], const floatx4 (&kf)[2], const floatx4 (&vf)[2],
                                           float qk_scale, bool masked, Hidden hidden, float down, SpState<INT8>& st,
                                           u32x4 (&pb)[MT]) {
  auto factor = [&](int e) { return INT8 ? kf[e >> 2][e & 3] : qk_scale; };
  float pr[MT][8], psum[MT];
  auto probs = [&]() {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pr[mt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][e >> 2][e & 3], factor(e), -st.m[mt]));
    if (masked) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 8; ++e) pr[mt][e] = hidden(mt, e) ? 0.f : pr[mt][e];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      psum[mt] = pr[mt][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) psum[mt] += pr[mt][e];
    }
  };
  probs();
  // (A row past the last has no reference, so its sum is infinite in a step without masks: a wave that holds one
  // takes the way below each time.)
  bool grow = INT8 && down != 1.f;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) grow |= psum[mt] > kSpLazy;
  if (__ballot(grow)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx = kNegBig;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, hidden(mt, e) ? kNegBig : s[mt][e >> 2][e & 3] * factor(e));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(st.m[mt], mx);
      float alpha = __builtin_amdgcn_exp2f(st.m[mt] - m_new);
      st.l[mt] *= alpha;
      if constexpr (INT8) alpha *= down;
#pragma unroll
      for (int j = 0; j < 8; ++j) st.o[mt][j] *= alpha;
      st.m[mt] = m_new;
    }
    probs();
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st.l[mt] += psum[mt];
    float(&x)[8] = pr[mt];
    if constexpr (INT8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= vf[e >> 2][e & 3];
      if (masked) {  // (a hidden key's value scale may be anything)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = hidden(mt, e) ? 0.f : x[e];
      }
      pb[mt] = u32x4{pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7])};
    } else {
      pb[mt] = u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
  }
}

// Two bf16 values with 0 in the place of those that are not finite; wild: there was one.
__device__ __forceinline__ uint32_t bf16x2_tame(uint32_t x, bool& wild) {
  const bool lo = (x & 0x7F80u) == 0x7F80u, hi = (x & 0x7F800000u) == 0x7F800000u;
  wild |= lo || hi;
  return (lo ? 0 : x & 0xFFFFu) | (hi ? 0 : x & 0xFFFF0000u);
}

// Exponent of a positive finite scale, as an integer power of two above it.
__device__ __forceinline__ int scale_exp(float x) { return (int)((__builtin_bit_cast(uint32_t, x) >> 23) & 0xFF) - 126; }
// 2^e by its bits, e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// A key's slot in the block that the table names, or in block 0 (and a flag) where it names none of the pool's.
__device__ __forceinline__ int sp_slot_in(const SpParams& p, int block, int key) {
  if (block < 0 || block >= p.num_blocks) {
    atomicOr(p.head, kErrBlock);
    block = 0;
  }
  return block * p.block_size + key % p.block_size;
}
__device__ __forceinline__ int sp_slot(const SpParams& p, const int32_t* bt, int key) { return sp_slot_in(p, bt[key / p.block_size], key); }

// ---- tiles ----
constexpr int kSpExpOff = kQtSlotOff + 2 * 8 * 4;  // int [2 buffers][2 waves]: the stage's largest value-scale exponents
constexpr int kSpLds = kSpExpOff + 2 * 2 * 4;

template <bool INT8, int SDT>
__device__ __forceinline__ void sp_tile_item(const SpParams& p, const SpItem& d, char* smem) {
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const bool of_group = d.kind == kGroupTile;
  const int head = d.head, seq = d.seq, rows_total = d.rows_total, row0 = d.row0, kstart = d.k0, kend = d.k1;
  const int first_seen = d.first_seen;
  const int64_t part_row = d.part_row + (int64_t)head * rows_total;
  const int kg_count = 256 / d.tile_rows;
  const int row_groups = kSpWaves / kg_count;
  const int r = lane & 15;
  const int g = lane >> 4;
  const int kg = wave / row_groups;
  const int wrow0 = row0 + (wave % row_groups) * kQtWaveRows;
  int* s_slot = (int*)(smem + kQtSlotOff);
  int* s_exp = (int*)(smem + kSpExpOff);
  const int32_t* bt = p.block_tables + (int64_t)seq * p.bt_stride;
  auto tile_slot = [&](int tile16) {
    return sp_slot(p, bt, min(kstart + kTileKeys * tile16, (kend - 1) & ~(kTileKeys - 1)));
  };
  int slot0 = 0;
  if (tid < 16) slot0 = tile_slot(tid);
  SpState<INT8> st;
  u32x4 raw[kQtMT][4];
  int kend_row[kQtMT], kend_wave = 0, kfull_wave = kend;
#pragma unroll
  for (int mt = 0; mt < kQtMT; ++mt) {
    const int row = wrow0 + kRows * mt + r;
    const bool valid = row < rows_total;
    const int t = valid ? row / p.group : 0;
    // (a row past the last reads the first token, a token past q the last one; neither is stored)
    const int token = min(of_group ? p.tokens[d.token + t] : d.token + t, p.num_rows - 1);
    kend_row[mt] = valid ? (of_group ? kend : min(kend, first_seen + t)) : 0;
    const uint16_t* src = p.q + (int64_t)token * p.q_tok_stride +
                          (int64_t)(head * p.group + (valid ? row - t * p.group : 0)) * p.q_head_stride + 8 * g;
#pragma unroll
    for (int c = 0; c < 4; ++c) raw[mt][c] = *(const u32x4*)(src + 32 * c);
  }
  if (wrow0 < rows_total) {
    const int last = (min(wrow0 + kQtWaveRows, rows_total) - 1) / p.group;
    kend_wave = of_group ? kend : min(kend, first_seen + last);
    kfull_wave = of_group ? kend : min(kend, first_seen + wrow0 / p.group);
  }
  if (tid < 16) s_slot[tid] = slot0;
  lds_barrier();  // (the query rows are still on their way)
  QtRegs<INT8> R;
  int vexp = -126;  // value scales are taken relative to 2^vexp
  auto stage_store = [&](int buf, int kb) {
    if constexpr (!INT8) {
      if (kb + kQtKeys > first_seen) {  // keys that some row does not see
        bool wild = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (kb + qt_octet_key(tid >> 5, e) < first_seen) continue;
          R.v[e][0] = bf16x2_tame(R.v[e][0], wild);
          R.v[e][1] = bf16x2_tame(R.v[e][1], wild);
        }
        if (wild) p.seqs[(int64_t)seq * kSpSeqInts + 9] = 1;
      }
    }
    qt_store_kv<INT8>(smem, buf, tid, R);
    if constexpr (INT8) {
      if (tid < 2 * kQtKeys) {
        float* sc = (float*)(smem + kQtScaleOff) + buf * 2 * kQtKeys;
        sc[tid] = tid < kQtKeys ? R.sc * p.qk_scale : R.sc;
        if (tid >= kQtKeys) {
          int x = fabsf(R.sc) < INFINITY ? scale_exp(R.sc) : -126;
#pragma unroll
          for (int o = 32; o >= 1; o >>= 1) x = max(x, __shfl_xor(x, o));
          if (lane == 0) s_exp[buf * 2 + wave - kQtKeys / kWave] = x;
        }
      }
    }
  };
  const int n_stages = (kend - kstart + kQtKeys - 1) / kQtKeys;
  qt_load<INT8, SDT>(p, s_slot, kstart, kend, head, tid, R);
  __asm__ __volatile__("" ::: "memory");  // the keys are requested before the query rows are waited for
#pragma unroll
  for (int mt = 0; mt < kQtMT; ++mt) {
#pragma unroll
    for (int c = 0; c < 4; ++c) st.q[mt].q[c] = sp_q_operand<INT8>(raw[mt][c]);
    st.m[mt] = kNegBig;
    st.l[mt] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[mt][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  stage_store(0, kstart);
  __syncthreads();
  for (int t = 0; t < n_stages; ++t) {
    const int buf = t & 1;
    const int kb0 = kstart + t * kQtKeys;
    const bool more = t + 1 < n_stages;
    int next_slot = 0;
    if (more) {
      qt_load<INT8, SDT>(p, s_slot + 8 * (buf ^ 1), kb0 + kQtKeys, kend, head, tid, R);
      if (tid < 8) next_slot = tile_slot(8 * (t + 2) + tid);
    }
    __asm__ __volatile__("" ::: "memory");  // the loads go out before the products
    float vscale = 1.f, down = 1.f;
    if constexpr (INT8) {
      if (kb0 + 32 * kg < kend_wave) {  // (a wave without a step here keeps its own power)
        const int x = max(__builtin_amdgcn_readfirstlane(max(s_exp[buf * 2], s_exp[buf * 2 + 1])), vexp);
        down = pow2(vexp - x);  // (2^-126 or less: what was added so far had scales that small)
        vexp = x;
      }
      vscale = pow2(-vexp);
    }
#pragma unroll 1
    for (int u = kg; u < 4; u += kg_count) {
      const int kb = kb0 + 32 * u;
      if (kb >= kend_wave) break;
      const bool masked = kb + 32 > kfull_wave;
      const char* ks = smem + buf * kQtStage;
      const char* vs = ks + kQtTileBytes;
      floatx4 s[kQtMT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int mt = 0; mt < kQtMT; ++mt) s[mt][h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4 a = *(const u32x4*)(ks + (32 * u + 16 * h + r) * 256 + qt_k_pos(r, 4 * c + g) * 16);
#pragma unroll
          for (int mt = 0; mt < kQtMT; ++mt) s[mt][h] = sp_mfma<INT8>(a, st.q[mt].q[c], s[mt][h]);
        }
      }
      floatx4 kf[2], vf[2];
      if constexpr (INT8) {
        const float* sc = (const float*)(smem + kQtScaleOff) + buf * 2 * kQtKeys + 32 * u + 4 * g;
        kf[0] = *(const floatx4*)sc;
        kf[1] = *(const floatx4*)(sc + 16);
        vf[0] = *(const floatx4*)(sc + kQtKeys) * vscale;
        vf[1] = *(const floatx4*)(sc + kQtKeys + 16) * vscale;
      }
      u32x4 pb[kQtMT];
      sp_softmax<INT8, kQtMT>(
          s, kf, vf, p.qk_scale, masked,
          [&](int mt, int e) { return kb + 16 * (e >> 2) + 4 * g + (e & 3) >= kend_row[mt]; }, down, st, pb);
      down = 1.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u32x4 a = *(const u32x4*)(vs + r * 256 + qt_v_pos(r, 4 * u + g) * 16 + j * 16 * 256);
#pragma unroll
        for (int mt = 0; mt < kQtMT; ++mt) {
          if constexpr (INT8)
            st.o[mt][j] = sp_mfma<true>(a, __builtin_bit_cast(f16x8, pb[mt]), st.o[mt][j]);
          else
            st.o[mt][j] = sp_mfma<false>(a, __builtin_bit_cast(bf16x8, pb[mt]), st.o[mt][j]);
        }
      }
    }
    if (more) {
      stage_store(buf ^ 1, kb0 + kQtKeys);
      if (tid < 8) s_slot[8 * buf + tid] = next_slot;
    }
    __syncthreads();
  }
  // ---- merge the key groups through LDS ----
#pragma unroll
  for (int mt = 0; mt < kQtMT; ++mt) {
    st.l[mt] += __shfl_xor(st.l[mt], 16);
    st.l[mt] += __shfl_xor(st.l[mt], 32);
    if constexpr (INT8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) st.o[mt][j] *= pow2(vexp);
    }
  }
  if (kg_count > 1) {
    floatx4* s_part = (floatx4*)smem;
    auto part_at = [&](int q, int mt, int j) -> floatx4& {
      return s_part[((((q - 1) * row_groups + wave % row_groups) * kQtMT + mt) * 9 + j) * kWave + lane];
    };
    // (KG - 1) * row groups is 6 for 64 rows, 4 for 128
    static_assert(6 * kQtMT * 9 * kWave * 16 <= kQtScaleOff, "partials fit the stages");
    if (kg > 0) {
#pragma unroll
      for (int mt = 0; mt < kQtMT; ++mt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) part_at(kg, mt, j) = st.o[mt][j];
        part_at(kg, mt, 8) = floatx4{st.m[mt], st.l[mt], 0.f, 0.f};
      }
    }
    __syncthreads();
    if (kg > 0) return;
    for (int q = 1; q < kg_count; ++q) {
#pragma unroll
      for (int mt = 0; mt < kQtMT; ++mt) {
        const floatx4 ml = part_at(q, mt, 8);
        const float mm = fmaxf(st.m[mt], ml[0]);
        const float a0 = __builtin_amdgcn_exp2f(st.m[mt] - mm);
        const float a1 = __builtin_amdgcn_exp2f(ml[0] - mm);
        st.l[mt] = a0 * st.l[mt] + a1 * ml[1];
        st.m[mt] = mm;
#pragma unroll
        for (int j = 0; j < 8; ++j) st.o[mt][j] = a0 * st.o[mt][j] + a1 * part_at(q, mt, j);
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < kQtMT; ++mt) {
    const int row = wrow0 + kRows * mt + r;
    if (row >= rows_total) continue;
    const int64_t to = part_row + row;
#pragma unroll
    for (int j = 0; j < 8; ++j) *(floatx4*)(p.part_o + to * kHeadDim + 16 * j + 4 * g) = st.o[mt][j];
    if (g == 0) *(float2*)(p.part_ml + to * 2) = float2{st.m[mt], st.l[mt]};
  }
}

// ---- light items ----
// A wave streams its KV head's tiles of 16 keys through a ring in LDS, copied by the memory system
// (no registers in flight), and holds one 32-key step in registers: the ring's two slots are
// requested again as soon as they are read.  Rows are swizzled in 16-byte chunks so that the
// fragment reads are free of conflicts.
template <bool INT8>
struct Light {
  static constexpr int kRowBytes = INT8 ? kHeadDim : 2 * kHeadDim;
  static constexpr int kTile = kTileKeys * kRowBytes;           // K (or V) of a tile
  static constexpr int kScale = INT8 ? 256 : 0;                 // key scales' dwords, then value scales'
  static constexpr int kSlot = 2 * kTile + kScale;
  static constexpr int kRing = INT8 ? 4 : 2;                    // tiles
  static constexpr int kCopies = 2 * kTile / 1024 + (INT8 ? 1 : 0);  // copy instructions per tile
  static constexpr int kChunks = kRowBytes / 16;                // per row
};
constexpr int kLightWindow = 512;  // tiles whose slots a wave lists at a time
constexpr int kLightWaveBytes = Light<true>::kRing * Light<true>::kSlot;
static_assert(Light<false>::kRing * Light<false>::kSlot <= kLightWaveBytes, "a wave's ring");
constexpr int kLightSlotOff = kSpWaves * kLightWaveBytes;  // int [waves][kLightWindow]
constexpr int kLightScaleOff = kLightSlotOff + kSpWaves * kLightWindow * 4;  // float [waves][64]
constexpr int kLightLds = kLightScaleOff + kSpWaves * kWave * 4;
static_assert(kLightLds <= 160 * 1024, "LDS of one CU");

template <int BYTES>
__device__ __forceinline__ void copy_to_lds(const void* src, void* lds) {
  static_assert(BYTES == 16 || BYTES == 4, "bytes per lane");
  if constexpr (BYTES == 16)
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
  else
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)lds, 4, 0, 0);
}
// s_waitcnt with only vmcnt or only lgkmcnt (0) constrained
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }
// At most the copies of the n newest tiles (0 .. 2) still in flight.
template <int PER>
__device__ __forceinline__ void wait_tiles(int n) {
  if (n <= 0)
    wait_vmcnt<0>();
  else if (n == 1)
    wait_vmcnt<PER>();
  else
    wait_vmcnt<2 * PER>();
}

// A 32-key step in registers: K chunk c of tile t holds dims 32 g + 8 c .. of key r (int8: bytes of
// two chunks in one vector); V slot e dims 8 r .. of key 16 (e / 4) + 4 g + e % 4.
template <bool INT8>
struct LightRegs;
template <>
struct LightRegs<true> {
  u32x4 k[2][2];
  u32x2 v[8];
};
template <>
struct LightRegs<false> {
  u32x4 k[2][4];
  u32x4 v[8];
};

template <bool INT8, int SDT, int MT>
__device__ __forceinline__ void sp_light(const SpParams& p, const SpItem& d, int head, int kstart0, int kend0, int64_t part_row, char* smem) {
  using L = Light<INT8>;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lane = tid % kWave;
  const int r = lane & 15, g = lane >> 4;
  const int seq = d.seq, rows_total = d.rows_total, first_seen = d.first_seen;
  const int32_t* bt = p.block_tables + (int64_t)seq * p.bt_stride;
  char* ring = smem + wave * kLightWaveBytes;
  int* s_slot = (int*)(smem + kLightSlotOff) + wave * kLightWindow;
  float* s_sc = (float*)(smem + kLightScaleOff) + wave * kWave;
  const int64_t slot_bytes = (int64_t)p.num_kv_heads * L::kRowBytes;
  // this lane's part of a copy: key, and chunk position
  constexpr int kPerCopy = 1024 / L::kRowBytes;  // keys per copy
  const int copy_key = lane / L::kChunks, copy_pos = lane % L::kChunks;
  auto copy_tile = [&](int t) {  // tile t of the window
    const int64_t slot0 = __builtin_amdgcn_readfirstlane(s_slot[t]);
    char* dst = ring + (t % L::kRing) * L::kSlot;
    const char* kc = (const char*)p.k_cache + slot0 * slot_bytes + (int64_t)head * L::kRowBytes;
    const char* vc = (const char*)p.v_cache + slot0 * slot_bytes + (int64_t)head * L::kRowBytes;
#pragma unroll
    for (int j = 0; j < L::kTile / 1024; ++j) {
      const int key = j * kPerCopy + copy_key;
      const uint32_t off = (uint32_t)key * (uint32_t)slot_bytes + 16u * (uint32_t)(copy_pos ^ (key & (L::kChunks - 1)));
      copy_to_lds<16>(kc + off, dst + j * 1024);
      copy_to_lds<16>(vc + off, dst + L::kTile + j * 1024);
    }
    if constexpr (INT8) {
      // lanes 0..15: the dwords that hold the keys' scales, 16..31 the values' (the rest repeat them)
      const int64_t at = (slot0 + (lane & 15)) * p.num_kv_heads + head;
      copy_to_lds<4>((const char*)((lane & 16) ? p.v_scale : p.k_scale) + (at & ~1ll) * 2, dst + 2 * L::kTile);
    }
  };
  // the first slots and the query rows, requested together
  const int key0 = min(kstart0 + kTileKeys * lane, (kend0 - 1) & ~(kTileKeys - 1));
  const int block0 = bt[key0 / p.block_size];
  SpState<INT8> st;
  u32x4 raw[MT][4];
  int kend_row[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = kRows * mt + r;
    const bool valid = row < rows_total;
    const int t = valid ? row / p.group : 0;
    kend_row[mt] = valid ? min(kend0, first_seen + t) : 0;
    const uint16_t* src = p.q + (int64_t)min(d.token + t, p.num_rows - 1) * p.q_tok_stride +
                          (int64_t)(head * p.group + (valid ? row - t * p.group : 0)) * p.q_head_stride + 32 * g;
#pragma unroll
    for (int c = 0; c < 4; ++c) raw[mt][c] = *(const u32x4*)(src + 8 * c);
  }
  const int slot0 = sp_slot_in(p, block0, key0);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int c = 0; c < 4; ++c) st.q[mt].q[c] = sp_q_operand<INT8>(raw[mt][c]);
    st.m[mt] = kNegBig;
    st.l[mt] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[mt][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  int vexp = -126;
  const int kfull = min(kend0, first_seen);
  for (int kstart = kstart0; kstart < kend0; kstart += kLightWindow * kTileKeys) {
    const int kend = min(kend0, kstart + kLightWindow * kTileKeys);
    const int n_tiles = (kend - kstart + kTileKeys - 1) / kTileKeys;
    const int n_steps = (n_tiles + 1) / 2;
    for (int t = lane; t < n_tiles; t += kWave) s_slot[t] = t < kWave && kstart == kstart0 ? slot0 : sp_slot(p, bt, kstart + kTileKeys * t);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < L::kRing; ++t)
      if (t < n_tiles) copy_tile(t);
#pragma unroll 1
    for (int it = 0; it < n_steps; ++it) {
      const int kb = kstart + 32 * it;
      const bool masked = kb + 32 > kfull;
      wait_tiles<L::kCopies>(min(n_tiles, 2 * it + L::kRing) - (2 * it + 2));
      LightRegs<INT8> R;
      float sc = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char* sl = ring + ((2 * it + t) % L::kRing) * L::kSlot;
        if constexpr (INT8) {
          R.k[t][0] = *(const u32x4*)(sl + r * 128 + ((2 * g) ^ (r & 7)) * 16);
          R.k[t][1] = *(const u32x4*)(sl + r * 128 + ((2 * g + 1) ^ (r & 7)) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 4 * g + i;
            R.v[4 * t + i] = *(const u32x2*)(sl + L::kTile + key * 128 + ((r >> 1) ^ (key & 7)) * 16 + (r & 1) * 8);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) R.k[t][c] = *(const u32x4*)(sl + r * 256 + ((4 * g + c) ^ r) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 4 * g + i;
            R.v[4 * t + i] = *(const u32x4*)(sl + L::kTile + key * 256 + (r ^ key) * 16);
          }
        }
      }
      if constexpr (INT8) {
        // lanes 0..31: key scale of key lane; 32..63: value scale of key lane - 32
        const int key = lane & 31;
        const char* sl = ring + ((2 * it + (key >> 4)) % L::kRing) * L::kSlot + 2 * L::kTile;
        const uint32_t two = *(const uint32_t*)(sl + ((lane >> 5) * 16 + (key & 15)) * 4);
        const int64_t at = (int64_t)(key & 15) * p.num_kv_heads + head;  // (a tile's first slot is even)
        const uint16_t raw = (uint16_t)((at & 1) ? two >> 16 : two);
        sc = SDT == NE_DTYPE_BF16 ? bf16_to_f32(raw) : f16_to_f32(raw);
        sc = kb + key < kend ? sc : 0.f;  // a slot past the end may hold anything
      }
      wait_lgkmcnt0();  // the two slots are read: request them again
      if (2 * it + L::kRing < n_tiles) copy_tile(2 * it + L::kRing);
      if (2 * it + 1 + L::kRing < n_tiles) copy_tile(2 * it + 1 + L::kRing);
      floatx4 s[MT][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4 a;
          if constexpr (INT8)
            a = i8x8_f16x8(R.k[t][c >> 1][2 * (c & 1)], R.k[t][c >> 1][2 * (c & 1) + 1]);
          else
            a = R.k[t][c];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) s[mt][t] = sp_mfma<INT8>(a, st.q[mt].q[c], s[mt][t]);
        }
      }
      floatx4 kf[2], vf[2];
      float down = 1.f;
      if constexpr (INT8) {
        const int ex = lane >= 32 && fabsf(sc) < INFINITY ? scale_exp(sc) : -126;
        if (__ballot(ex > vexp)) {  // a larger value scale than so far
          int top = ex;
#pragma unroll
          for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o));
          top = __builtin_amdgcn_readfirstlane(top);
          down = pow2(vexp - top);
          vexp = top;
        }
        s_sc[lane] = sc * (lane < 32 ? p.qk_scale : pow2(-vexp));
        __builtin_amdgcn_wave_barrier();
        kf[0] = *(const floatx4*)(s_sc + 4 * g);
        kf[1] = *(const floatx4*)(s_sc + 16 + 4 * g);
        vf[0] = *(const floatx4*)(s_sc + 32 + 4 * g);
        vf[1] = *(const floatx4*)(s_sc + 48 + 4 * g);
        __builtin_amdgcn_wave_barrier();
      }
      u32x4 pb[MT];
      sp_softmax<INT8, MT>(
          s, kf, vf, p.qk_scale, masked,
          [&](int mt, int e) { return kb + 16 * (e >> 2) + 4 * g + (e & 3) >= kend_row[mt]; }, down, st, pb);
      if constexpr (!INT8) {
        if (masked) {
          // values past the end may be stale bits; one that some row does not see must not reach that row
          bool wild = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = kb + 16 * (e >> 2) + 4 * g + (e & 3);
            if (key >= kend) R.v[e] = u32x4{0, 0, 0, 0};
            if (key < first_seen) continue;
#pragma unroll
            for (int w = 0; w < 4; ++w) R.v[e][w] = bf16x2_tame(R.v[e][w], wild);
          }
          if (wild) p.seqs[(int64_t)seq * kSpSeqInts + 9] = 1;
        }
      }
      {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u32x4 a;
          if constexpr (INT8) {
            uint32_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = R.v[e][j >> 2];
            a = (j & 3) == 0   ? i8_cols_f16x8<0>(x)
                : (j & 3) == 1 ? i8_cols_f16x8<1>(x)
                : (j & 3) == 2 ? i8_cols_f16x8<2>(x)
                               : i8_cols_f16x8<3>(x);
          } else {
            const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
            a = u32x4{__builtin_amdgcn_perm(R.v[1][j >> 1], R.v[0][j >> 1], sel), __builtin_amdgcn_perm(R.v[3][j >> 1], R.v[2][j >> 1], sel),
                      __builtin_amdgcn_perm(R.v[5][j >> 1], R.v[4][j >> 1], sel), __builtin_amdgcn_perm(R.v[7][j >> 1], R.v[6][j >> 1], sel)};
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if constexpr (INT8)
              st.o[mt][j] = sp_mfma<true>(a, __builtin_bit_cast(f16x8, pb[mt]), st.o[mt][j]);
            else
              st.o[mt][j] = sp_mfma<false>(a, __builtin_bit_cast(bf16x8, pb[mt]), st.o[mt][j]);
          }
        }
      }
    }
  }
  wait_vmcnt<0>();  // no copy lands in LDS after the wave has left
  const float back = INT8 ? pow2(vexp) : 1.f;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int row = kRows * mt + r;
    float l = st.l[mt];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (row >= rows_total) continue;
    const int64_t to = part_row + (int64_t)head * rows_total + row;
    float* po = p.part_o + to * kHeadDim + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *(floatx4*)(po + 8 * i) = floatx4{st.o[mt][0][i], st.o[mt][1][i], st.o[mt][2][i], st.o[mt][3][i]} * back;
      *(floatx4*)(po + 8 * i + 4) = floatx4{st.o[mt][4][i], st.o[mt][5][i], st.o[mt][6][i], st.o[mt][7][i]} * back;
    }
    if (g == 0) *(float2*)(p.part_ml + to * 2) = float2{st.m[mt], l};
  }
}

constexpr int kSpAllLds = kSpLds > kLightLds ? kSpLds : kLightLds;

template <bool INT8, int SDT>
__global__ __launch_bounds__(kSpThreads) void shared_prefix_parts_kernel(SpParams p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // the item is requested beside the count that says whether there is one
  SpItem d;
  const ConstI32* src = (const ConstI32*)(p.items + blockIdx.x);
#pragma unroll
  for (int i = 0; i < 14; ++i) ((int32_t*)&d)[i] = src[i];
  if ((int)blockIdx.x >= ((const ConstI32*)p.head)[1]) return;
  if (d.kind != kLight) {
    sp_tile_item<INT8, SDT>(p, d, smem);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int part = d.part0 + wave / p.light_heads;
  const int head = d.head + wave % p.light_heads;
  if (wave >= p.light_heads * p.light_keys || part >= d.parts || head >= p.num_kv_heads) return;  // (no barrier follows)
  const int k0 = d.k0 + (int)((int64_t)d.tiles * part / d.parts) * kTileKeys;
  const int k1 = min(d.k0 + (int)((int64_t)d.tiles * (part + 1) / d.parts) * kTileKeys, d.k1);
  const int64_t row = d.part_row + (int64_t)part * p.num_kv_heads * d.rows_total;
  if (d.rows_total <= kRows)
    sp_light<INT8, SDT, 1>(p, d, head, k0, k1, row, smem);
  else
    sp_light<INT8, SDT, 2>(p, d, head, k0, k1, row, smem);
}

// ---- merge ----
constexpr int kMergeThreads = 256;
constexpr int kMergeAhead = 8;
// Up to this many rows, which then have many parts each, 64 threads take a row's parts in turn: 320 rows of 63
// parts 12.5 to 6 us; 1,280 rows of few parts would take 0.7 us longer.
constexpr int kMergeFewRows = 1024;

template <int LANES>
__global__ __launch_bounds__(kMergeThreads) void shared_prefix_merge_kernel(SpParams p, int blocks_per_seq) {
  const int seq = blockIdx.x / blocks_per_seq;
  const ConstI32* d = (const ConstI32*)(p.seqs + (int64_t)seq * kSpSeqInts);
  const int heads = p.num_kv_heads * p.group;
  const int x = (blockIdx.x % blocks_per_seq) * (kMergeThreads / LANES) + (int)threadIdx.x / LANES;  // query, then head
  if (x >= d[0] * heads) return;
  if (d[1] > p.num_rows - d[0]) {  // the plan was made for more rows than q has
    if (threadIdx.x == 0) atomicOr(p.head, kErrRows);
    return;
  }
  const int i = x / heads, head = x % heads;
  const int kv = head / p.group, in = i * p.group + head % p.group;
  const int np = d[2], n = np + d[3];
  const int64_t prefix0 = d[4] + kv * d[5] + in, own0 = d[6] + kv * d[7] + in;
  const int64_t prefix_step = p.num_kv_heads * d[5], own_step = p.num_kv_heads * d[7];
  const int cd = (threadIdx.x & 15) * 8;
  constexpr int kTurns = LANES / 16;  // sets of 16 lanes that take parts in turn
  const int turn = (int)threadIdx.x % LANES / 16;
  float M = kNegBig, L = 0.f;
  float acc[8] = {};
  for (int s0 = turn; s0 < n; s0 += kMergeAhead * kTurns) {
    float2 ml[kMergeAhead];
    floatx4 a[kMergeAhead], b[kMergeAhead];
#pragma unroll
    for (int j = 0; j < kMergeAhead; ++j) {
      const int s = min(s0 + j * kTurns, n - 1);
      const int64_t row = s < np ? prefix0 + s * prefix_step : own0 + (s - np) * own_step;
      ml[j] = *(const float2*)(p.part_ml + row * 2);
      a[j] = *(const floatx4*)(p.part_o + row * kHeadDim + cd);
      b[j] = *(const floatx4*)(p.part_o + row * kHeadDim + cd + 4);
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < kMergeAhead; ++j) top = fmaxf(top, s0 + j * kTurns < n ? ml[j].x : kNegBig);
    const float down = __builtin_amdgcn_exp2f(M - top);
    L *= down;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] *= down;
    M = top;
#pragma unroll
    for (int j = 0; j < kMergeAhead; ++j) {
      if (s0 + j * kTurns >= n) continue;
      const float w = __builtin_amdgcn_exp2f(ml[j].x - M);
      L += w * ml[j].y;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[c] += w * a[j][c];
        acc[c + 4] += w * b[j][c];
      }
    }
  }
#pragma unroll
  for (int o = 16; o < LANES; o <<= 1) {  // the sets' sums, the same in each
    const float top = fmaxf(M, __shfl_xor(M, o)), down = __builtin_amdgcn_exp2f(M - top);
    M = top;
    L *= down;
    L += __shfl_xor(L, o);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      acc[c] *= down;
      acc[c] += __shfl_xor(acc[c], o);
    }
  }
  if (d[9]) {  // values that are not finite, of keys that only some rows see: this row's
    const int last = min(d[8] - d[0] + i, min(d[8], p.max_ctx) - 1);  // the last key it sees
    for (int key = max(d[8] - d[0] + 1, 0); key <= last && key / p.block_size < p.bt_stride; ++key) {
      const int64_t slot = sp_slot(p, p.block_tables + (int64_t)seq * p.bt_stride, key);
      const uint16_t* v = (const uint16_t*)p.v_cache + (slot * p.num_kv_heads + kv) * kHeadDim + cd;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float x = bf16_to_f32(v[c]);
        acc[c] += fabsf(x) < INFINITY ? 0.f : x;
      }
    }
  }
  if (turn != 0) return;
  // a row that sees no key is zero
  const bool none = L == 0.f;
  const float inv = none ? 0.f : 1.f / L;
  uint16_t* to = p.out + (int64_t)(d[1] + i) * p.o_tok_stride + (int64_t)head * p.o_head_stride + cd;
  *(u32x4*)to = none ? u32x4{0, 0, 0, 0}
                     : u32x4{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                             pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv)};
}

// ---- host ----
struct SpLayout {
  int max_items, light_heads, light_keys, head_blocks;
  int64_t part_rows;
  size_t tokens, items, seqs, part_o, part_ml, total;
};

// Bounds that hold for any lengths within the call's (comments give the plan's counts).
SpLayout sp_layout(int num_seqs, int num_groups, int num_q_heads, int num_kv_heads, int max_q, int max_ctx, int max_prefix) {
  SpLayout l;
  const int group = num_q_heads / num_kv_heads;
  const int64_t tokens = (int64_t)num_seqs * max_q;
  const int64_t rows = tokens * group;
  if (max_prefix > max_ctx) max_prefix = max_ctx;
  l.light_heads = num_kv_heads < kSpWaves ? num_kv_heads : kSpWaves;
  l.light_keys = kSpWaves / l.light_heads;
  l.head_blocks = cdiv(num_kv_heads, l.light_heads);
  // Items: one per (tile, KV head) and one per (sequence, head block), and those of further parts: n stages,
  // or 16-key tiles, are cut into n / each parts, rounded, so there are less than n / each further ones;
  // `each` is worth a kNumCu-th of all work at least, so they are kNumCu in all (a few more by rounding),
  // and n - 1 of each n at most.
  const int64_t groups = max_prefix >= kTileKeys ? (num_groups < num_seqs / 2 ? num_groups : num_seqs / 2) : 0;
  const bool heavy = (int64_t)max_q * group > kLightRows;
  const int64_t light_rows = max_q * group < kLightRows ? max_q * group : kLightRows;
  int64_t items = (int64_t)num_seqs * l.head_blocks, part_rows = num_seqs * light_rows * num_kv_heads, further = 0, further_rows = 0;
  auto add_tiles = [&](int64_t tiles, int64_t stages) {
    items += tiles * num_kv_heads;
    part_rows += rows * num_kv_heads;
    further += tiles * (stages - 1) * num_kv_heads;
    further_rows += rows * (stages - 1) * num_kv_heads;
  };
  if (groups > 0) add_tiles(rows / 128 + groups, cdiv(max_prefix, kQtKeys));
  if (heavy) add_tiles(rows / 128 + num_seqs, cdiv(max_ctx, kQtKeys));
  const int64_t splits = (cdiv(max_ctx, kTileKeys) + kLightMinTiles / 2) / kLightMinTiles;  // of one sequence
  const int64_t light_further = num_seqs * (splits > 1 ? splits - 1 : 0);  // waves' parts
  further += light_further * l.head_blocks;
  further_rows += light_further * light_rows * num_kv_heads;
  const int64_t most = kNumCu + 16;
  items += further < most ? further : most;
  // a further part of a tile has up to 256 rows of one head; of a light item light_rows of its heads, for each of its waves' parts
  const int64_t per = 256 > light_rows * l.light_heads * l.light_keys ? 256 : light_rows * l.light_heads * l.light_keys;
  part_rows += further_rows < most * per ? further_rows : most * per;
  l.part_rows = part_rows;
  l.max_items = (int)items;
  size_t at = 256;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.tokens = take((size_t)(tokens + 1) * 4);
  l.items = take((size_t)l.max_items * sizeof(SpItem));
  l.seqs = take((size_t)num_seqs * kSpSeqInts * 4);
  l.part_ml = take((size_t)l.part_rows * 8);
  l.part_o = take((size_t)l.part_rows * kHeadDim * 4);
  l.total = at;
  return l;
}

bool sp_shape_ok(int num_seqs, int num_groups, int num_q_heads, int num_kv_heads, int max_q, int max_ctx) {
  return num_seqs >= 1 && num_seqs <= kSpMaxSeqs && num_groups >= 0 && num_groups <= num_seqs && num_kv_heads >= 1 &&
         num_kv_heads <= 256 && num_q_heads >= num_kv_heads && num_q_heads % num_kv_heads == 0 && num_q_heads <= 4096 &&
         max_q >= 1 && max_ctx >= 1 && max_ctx <= (1 << 30) && (int64_t)num_seqs * max_q * num_q_heads < (1ll << 30);
}

int sp_check(const char* what, int num_seqs, int num_groups, int num_q_heads, int num_kv_heads, int max_q, int max_ctx, int max_prefix,
             int block_size, int num_blocks, int bt_stride, const void* ws, size_t bytes, SpLayout& l) {
  NE_CHECK_ARG(num_seqs >= 0 && num_groups >= 0 && num_groups <= num_seqs, "%s: bad sizes: %d sequences, %d groups", what, num_seqs, num_groups);
  NE_CHECK_SUPPORTED(num_seqs <= kSpMaxSeqs, "%s: %d sequences exceed %d", what, num_seqs, kSpMaxSeqs);
  NE_CHECK_ARG(sp_shape_ok(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q, max_ctx),
               "%s: bad shape: %d / %d heads, %d queries, %d keys", what, num_q_heads, num_kv_heads, max_q, max_ctx);
  NE_CHECK_ARG(max_prefix >= 0, "%s: bad prefix bound %d", what, max_prefix);
  NE_CHECK_SUPPORTED(block_size >= kTileKeys && block_size % kTileKeys == 0, "%s: block_size %d is not a multiple of 16", what, block_size);
  NE_CHECK_ARG(num_blocks >= 1 && (int64_t)num_blocks * block_size < (1ll << 31), "%s: bad pool of %d blocks", what, num_blocks);
  NE_CHECK_ARG(bt_stride >= 0, "%s: bad block table stride %d", what, bt_stride);
  NE_CHECK_ARG(ws, "%s: null workspace", what);
  NE_CHECK_ARG((uintptr_t)ws % 16 == 0, "%s: workspace must be 16-byte aligned", what);
  l = sp_layout(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q, max_ctx, max_prefix);
  NE_CHECK_SUPPORTED(l.part_rows < (1ll << 31), "%s: %lld rows of partial sums", what, (long long)l.part_rows);
  if (bytes < l.total) {
    set_error("%s: workspace of %zu bytes, %zu needed", what, bytes, l.total);
    return NE_EWORKSPACE;
  }
  return NE_OK;
}

void sp_bind(SpParams& p, const SpLayout& l, char* ws) {
  p.head = (uint32_t*)ws;
  p.tokens = (int32_t*)(ws + l.tokens);
  p.items = (SpItem*)(ws + l.items);
  p.seqs = (int32_t*)(ws + l.seqs);
  p.part_o = (float*)(ws + l.part_o);
  p.part_ml = (float*)(ws + l.part_ml);
  p.max_items = l.max_items;
  p.light_heads = l.light_heads;
  p.light_keys = l.light_keys;
  p.head_blocks = l.head_blocks;
  p.part_rows = l.part_rows;
}

template <bool INT8, int SDT>
int sp_launch(const SpParams& p, hipStream_t s) {
  static const hipError_t attr = hipFuncSetAttribute((const void*)shared_prefix_parts_kernel<INT8, SDT>,
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, kSpAllLds);
  if (attr != hipSuccess) {
    set_error("shared_prefix_parts: cannot reserve %d bytes of LDS: %s", kSpAllLds, hipGetErrorString(attr));
    return NE_ELAUNCH;
  }
  hipLaunchKernelGGL((shared_prefix_parts_kernel<INT8, SDT>), dim3(p.max_items), dim3(kSpThreads), kSpAllLds, s, p);
  const int rc = check_launch("shared_prefix_parts");
  if (rc != NE_OK) return rc;
  const int rows = p.max_q * p.num_kv_heads * p.group;
  const bool few = p.num_seqs * rows <= kMergeFewRows;
  const int per_seq = cdiv(rows, kMergeThreads / (few ? 64 : 16));
  hipLaunchKernelGGL(few ? shared_prefix_merge_kernel<64> : shared_prefix_merge_kernel<16>, dim3(p.num_seqs * per_seq), dim3(kMergeThreads), 0, s, p,
                     per_seq);
  return check_launch("shared_prefix_merge");
}

}  // namespace

}  // namespace ne

extern "C" size_t ne_shared_prefix_workspace_size(int32_t num_seqs, int32_t num_groups, int32_t num_q_heads,
                                                  int32_t num_kv_heads, int32_t max_q_len, int32_t max_ctx_len,
                                                  int32_t max_prefix_len) {
  if (!ne::sp_shape_ok(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len, max_ctx_len) || max_prefix_len < 0) return 0;
  return ne::sp_layout(num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len, max_ctx_len, max_prefix_len).total;
}

extern "C" int ne_shared_prefix_plan(const int32_t* ctx_len, const int32_t* q_start, const int32_t* q_len, int32_t num_rows,
                                     const int32_t* group_seqs, const int32_t* group_start, const int32_t* prefix_len,
                                     int32_t num_seqs, int32_t num_groups, int32_t num_q_heads, int32_t num_kv_heads,
                                     int32_t max_q_len, int32_t max_ctx_len, int32_t max_prefix_len, int32_t block_table_stride,
                                     int32_t block_size, int32_t num_blocks, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  using namespace ne;
  if (num_seqs == 0) return NE_OK;
  SpLayout l;
  const int rc = sp_check("shared_prefix_plan", num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len, max_ctx_len,
                          max_prefix_len, block_size, num_blocks, block_table_stride, workspace, workspace_bytes, l);
  if (rc != NE_OK) return rc;
  NE_CHECK_ARG(ctx_len && q_start && q_len && group_seqs && group_start && (prefix_len || num_groups == 0),
               "null pointer argument");
  NE_CHECK_ARG(num_rows >= 0, "bad row count %d", num_rows);
  SpParams p;
  memset(&p, 0, sizeof(p));
  sp_bind(p, l, (char*)workspace);
  p.ctx_len = ctx_len;
  p.q_start = q_start;
  p.q_len = q_len;
  p.group_seqs = group_seqs;
  p.group_start = group_start;
  p.prefix_len = prefix_len;
  p.num_rows = num_rows;
  p.num_seqs = num_seqs;
  p.num_groups = num_groups;
  p.num_kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_q = max_q_len;
  // a prefix longer than its bound is read as own keys past it
  p.max_ctx = max_ctx_len;
  p.bt_stride = block_table_stride;
  p.block_size = block_size;
  const int threads = cdiv(num_seqs < 256 ? 256 : num_seqs, kWave) * kWave;  // one per sequence
  hipLaunchKernelGGL(shared_prefix_plan_kernel, dim3(1), dim3(threads), 0, (hipStream_t)stream, p, max_prefix_len);
  return check_launch("shared_prefix_plan");
}

extern "C" int ne_shared_prefix_attention_rows(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t num_rows,
                                               const void* k_cache, const void* v_cache, const void* k_scale,
                                               const void* v_scale, int32_t kv_dtype, int32_t scale_dtype,
                                               const int32_t* block_tables, int32_t block_table_stride, int32_t block_size,
                                               int32_t num_blocks, int32_t num_seqs, int32_t num_groups, int32_t num_q_heads,
                                               int32_t num_kv_heads, int32_t head_dim, int32_t max_q_len, int32_t max_ctx_len,
                                               int32_t max_prefix_len, float softmax_scale, void* out,
                                               int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                               size_t workspace_bytes, void* stream) {
  using namespace ne;
  NE_CHECK_ARG(num_rows >= 0, "shared_prefix_attention: bad row count %d", num_rows);
  if (num_seqs == 0 || num_rows == 0) return NE_OK;
  NE_CHECK_SUPPORTED(head_dim == kHeadDim, "head_dim %d: only 128 is supported", head_dim);
  SpLayout l;
  const int rc = sp_check("shared_prefix_attention", num_seqs, num_groups, num_q_heads, num_kv_heads, max_q_len, max_ctx_len,
                          max_prefix_len, block_size, num_blocks, block_table_stride, workspace, workspace_bytes, l);
  if (rc != NE_OK) return rc;
  NE_CHECK_ARG(q && k_cache && v_cache && block_tables && out, "null pointer argument");
  NE_CHECK_ARG(kv_dtype == NE_DTYPE_BF16 || kv_dtype == NE_DTYPE_INT8, "the cache must be bf16 or int8");
  NE_CHECK_ARG(softmax_scale == softmax_scale, "softmax_scale is NaN");
  const bool int8 = kv_dtype == NE_DTYPE_INT8;
  if (int8) {
    NE_CHECK_ARG(k_scale && v_scale, "int8 cache needs scales");
    NE_CHECK_ARG(scale_dtype == NE_DTYPE_BF16 || scale_dtype == NE_DTYPE_FP16, "scales must be bf16 or fp16");
    NE_CHECK_ARG(((uintptr_t)k_scale | (uintptr_t)v_scale) % 4 == 0, "scales must be 4-byte aligned");
  }
  NE_CHECK_ARG(((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                   (q_token_stride | q_head_stride | out_token_stride | out_head_stride) % 8 == 0,
               "q, out and the caches must be 16-byte aligned, row and head strides multiples of 8 elements");
  SpParams p;
  memset(&p, 0, sizeof(p));
  sp_bind(p, l, (char*)workspace);
  p.q = (const uint16_t*)q;
  p.q_tok_stride = q_token_stride;
  p.q_head_stride = q_head_stride;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.num_seqs = num_seqs;
  p.num_groups = num_groups;
  p.num_rows = num_rows;
  p.num_kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_q = max_q_len;
  p.max_ctx = max_ctx_len;
  p.qk_scale = softmax_scale * kLog2e;
  p.out = (uint16_t*)out;
  p.o_tok_stride = out_token_stride;
  p.o_head_stride = out_head_stride;
  if (!int8) return sp_launch<false, NE_DTYPE_BF16>(p, (hipStream_t)stream);
  return scale_dtype == NE_DTYPE_BF16 ? sp_launch<true, NE_DTYPE_BF16>(p, (hipStream_t)stream)
                                      : sp_launch<true, NE_DTYPE_FP16>(p, (hipStream_t)stream);
}

extern "C" int ne_shared_prefix_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_cache,
                                          const void* v_cache, const void* k_scale, const void* v_scale, int32_t kv_dtype,
                                          int32_t scale_dtype, const int32_t* block_tables, int32_t block_table_stride,
                                          int32_t block_size, int32_t num_blocks, int32_t num_seqs, int32_t num_groups,
                                          int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_q_len,
                                          int32_t max_ctx_len, int32_t max_prefix_len, float softmax_scale, void* out,
                                          int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  // as many rows as the plan was made for
  return ne_shared_prefix_attention_rows(q, q_token_stride, q_head_stride, 0x7FFFFFFF, k_cache, v_cache, k_scale, v_scale, kv_dtype,
                                         scale_dtype, block_tables, block_table_stride, block_size, num_blocks, num_seqs, num_groups,
                                         num_q_heads, num_kv_heads, head_dim, max_q_len, max_ctx_len, max_prefix_len, softmax_scale,
                                         out, out_token_stride, out_head_stride, workspace, workspace_bytes, stream);
}
