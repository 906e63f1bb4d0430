// Serving from a paged K/V cache: launch arguments, and what the kernels share -- which sequence a workgroup has, which rows and keys
// of it, and where those lie.
//
// A call has a ragged batch: sequence b has `L` tokens in the cache, the last `n` of them new, and its queries are n x group rows
// for each KV head (row r: new token r / group, query head r mod group of the KV head's group), so that a K/V tile is read once
// for all heads of a group.  Lengths, starts and page table lie on the device and may change between two replays of a captured launch:
// the host knows only how many sequences and new tokens there can be, lays a grid that suffices for any lengths, and every
// workgroup finds its place from the lengths themselves (find_place).
#pragma once
#include "ringattn_device.h"

namespace ringattn {
namespace paged {

constexpr int kKeyTile = 32;      // keys of a tile
constexpr int kFewRows = 32;      // query rows of a workgroup where a sequence's KV head has few of them (ringattn_paged_few.h)
constexpr int kManyRows = 256;    // ... and where it has many (ringattn_paged_many.h)
// Up to so many rows of a sequence's KV head are few.  Attention, us as few and as many, 32 heads on 8: 16 sequences of 4 K, 16 tokens each (64
// rows) 67 and 93, 24 tokens 126 and 96, 32 tokens 99 and 95, 40 tokens 203 and 94.  Weights, the same: 32 tokens 85 and 119, 48 tokens (192
// rows) 116 and 146; one of 32 K, 32 tokens 49 and 56, 48 tokens 64 and 69.
constexpr int kFewRowsMost = 64, kWeightFewRowsMost = 192;
// Of one sequence alone, whose row tiles make even runs: 24 tokens (96 rows) over 32 K 39 as few and 52 as many, over 100 K 122 and 122; 32 tokens 42 and
// 52, 133 and 123; 40 tokens 49 and 53, 155 and 124.
constexpr int kFewRowsAlone = 128;
// Of attention where there is little to do for all (ringattn_paged_fwd): us as many and as few, 32 heads on 8: four chunks of 64 over 1 K, 256 rows, 32
// key tiles a workgroup 26 and 17; one over 8 K, 64 tiles 32 and 27; of 128, 512 rows, 128 tiles 40 and 40; 16 chunks of 24 over 4 K, 96 rows,
// 187 tiles 109 and 127; four of 256 over 1 K, 1024 rows, 128 tiles 45 and 56.  8 heads, two chunks of 512 over 2 K, 64 tiles 34 and 23.
constexpr int kFewRowsMore = 512, kFewMore = 96;
constexpr int kFewWorkgroups = 256, kFewLeast = 16, kFewSmall = 32, kFewMerge = 16;     // see few_rows
constexpr int kManyWorkgroups = 256, kManyLeast = 8, kManySaved = 12, kMergeSharers = 4;  // see find_place, merge_many
constexpr int kFewSlots = 2 * kFewWorkgroups, kManySlots = 2 * kManyWorkgroups + 16;  // parts that there can be
constexpr int kManyKeys = 128;      // keys of a workgroup of paged_weights_kernel
constexpr int kWeightUnits = 2048;   // parts of rows that there can be, where it shares them out
constexpr int kMaxBatch = 4096;   // sequences of a call

struct Cache {
  char* k;              // [pages, kv_heads, page, D] by strides
  char* v;
  int64_t page_stride, head_stride;  // bytes
  int token_stride;                  // bytes
  int pages;            // of the pool: an entry of the table outside [0, pages) is a page that is not there
  const int* table;     // [batch, table_pages]
  int64_t table_stride;
  int table_pages, page_shift;
  const int* lens;      // [batch] tokens in the cache, the new ones among them
  const int* starts;    // [batch + 1] first new token of a sequence among all new ones
  int batch, tokens;    // sequences; new tokens at most (rows of q)
};

// What row tiles whose keys went to several workgroups leave to be put together.
struct Parts {
  float* o;       // sums of a part's rows
  float2* stat;   // their references (log2 units) and the sums of their weights
  int* arrived;   // few rows: how many parts of a row tile are there, [2 kFewWorkgroups]; 0 between launches
};

// Scores that are not the plain products (ringattn_paged_fwd_scored): a template parameter SC of the programs says which of these there are,
// 0 being plain scores; the masks of any scored call are data.
constexpr int kCapped = 1, kSloped = 2, kScored = 4;
struct Scoring {
  float cap_in, cap_out;  // x = scale q k log2(e) becomes c tanh(x / c), c = cap_out = cap log2(e): cap_in takes q k to 2 log2(e) x / c
  const float* slopes;    // [heads]
  const int* prefix;      // [batch]
  const int* first;       // [tokens]
};
// Scores of a 32 x 32 tile, as the products give them (lane (n, h): row n, keys key0 + 4 h + [0, 4) of every eight), to what the exponentials take
// a multiple of (score_unit), less a constant of all scores (score_base).  tanh y = 1 - 2 / (e^2y + 1): an exponential and a reciprocal, each off by
// 2^-23 of itself; the softmax takes -1 / (e^2y + 1) as it is, 2 c times that being the capped score less c, so that a cap costs four instructions
// a score.  An infinite score is the cap.
// In steps, so that none waits for the one before: each takes one score as far as the next stage (left to itself the compiler has each score's
// instructions one behind the other).  `at`: slope times dist.  Of a key that lies in front of its row a slope takes slope |dist| = -slope dist, so that
// what is added is at + slope (0, 1, 2, 3, 8, ...): no absolute values; keys behind their rows, which prefixes show, are put right after (turn_slopes).  The
// rounding of `at` is 2^-24 of slope times up to 27 more than the distance, also of the row's own key, whose sum is 0: 2^-19 of a slope.
template <int SC> constexpr int kShapeSteps = (SC & kCapped) ? ((SC & kSloped) ? 25 : 22) : (SC & kSloped) ? 16 : 0;
template <int SC> static __device__ __forceinline__ void shape_step(f32x16& s, int i, const Scoring& x, float unit, float slope, float at) {
  constexpr int kSlopeAt = (SC & kCapped) ? 9 : 0;
  if constexpr ((SC & kCapped) != 0) {
    if (i < 16) s[i] *= x.cap_in;
    if (i >= 2 && i < 18) s[i - 2] = __builtin_amdgcn_exp2f(s[i - 2]);
    if (i >= 5 && i < 21) s[i - 5] = -1.f - s[i - 5];
    if (i >= 6 && i < 22) s[i - 6] = __builtin_amdgcn_rcpf(s[i - 6]);
  }
  if constexpr ((SC & kSloped) != 0) {
    const int e = i - kSlopeAt;
    if (e >= 0 && e < 16) s[e] = __builtin_fmaf(s[e], unit, __builtin_fmaf(slope, (float)(8 * (e >> 2) + (e & 3)), at));
  }
}
// Scores of keys that lie behind their rows: slope dist has been added where it was to be taken.  per: of a score's own units.
static __device__ __forceinline__ void turn_slopes(f32x16& s, float slope, int dist, float per) {
  const float twice = -2.f * slope * per;
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf((float)max(dist + 8 * (e >> 2) + (e & 3), 0), twice, s[e]);
}
template <int SC> static __device__ __forceinline__ float shape_unit(const Scoring& x, float scale_log2) { return (SC & kCapped) ? 2.f * x.cap_out : scale_log2; }
// dist: key0 + 4 h less the row's place in the sequence.
template <int SC> static __device__ __forceinline__ void shape_scores(f32x16& s, const Scoring& x, float scale_log2, float slope, int dist) {
#pragma unroll
  for (int i = 0; i < kShapeSteps<SC>; ++i) {
    shape_step<SC>(s, i, x, shape_unit<SC>(x, scale_log2), slope, slope * (float)dist);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <int SC> static __device__ __forceinline__ float score_unit(const Scoring& x, float scale_log2) {
  return (SC & kSloped) ? 1.f : shape_unit<SC>(x, scale_log2);
}
template <int SC> static __device__ __forceinline__ float score_base(const Scoring& x) { return (SC & kCapped) ? x.cap_out : 0.f; }

struct AttendArgs {
  Cache c;
  Scoring x;
  const char* q;
  char* out;
  float* lse;             // [heads, tokens]
  int64_t q_ts, q_hs, o_ts, o_hs;  // bytes between tokens, between heads
  int kv_heads, group;
  Divisor by_group, by_kv_heads;
  float scale_log2;
  int causal, window, sinks;
  int out_fp32;
  int few_most;           // rows of a sequence's KV head up to which it has few
  int many_cut;           // whether key tiles are shared out where there are many rows
  int few_shift;          // few rows: key tiles are dealt out 2^few_shift at a time, so that 2^30 suffice
  int few_begin;          // workgroups [few_begin, few_begin + kFewWorkgroups) have the sequences of few rows, the others those of many
  Parts few, many;
};

struct Seq {
  int len, start, n;
  int prefix;  // tokens at the beginning that every new one sees (0 but for scored calls)
};
static __device__ __forceinline__ int clamped(int x, int lo, int hi) { return min(max(x, lo), hi); }
// Lengths are data: whatever they hold, nothing outside the tensors is touched.  (A sequence's own are held to its table and to the call's tokens
// here; few_rows looks at what starts that do not ascend make of them all together.)
static __device__ __forceinline__ Seq seq_of(const Cache& c, int b, const int* prefix = nullptr) {
  Seq s;
  s.len = clamped(c.lens[b], 0, c.table_pages << c.page_shift);
  s.start = clamped(c.starts[b], 0, c.tokens);
  s.n = clamped(c.starts[b + 1], s.start, c.tokens) - s.start;
  s.prefix = prefix ? clamped(prefix[b], 0, s.len) : 0;
  return s;
}

static __device__ __forceinline__ Seq uniform(const Seq& s) {
  return Seq{__builtin_amdgcn_readfirstlane(s.len), __builtin_amdgcn_readfirstlane(s.start), __builtin_amdgcn_readfirstlane(s.n),
             __builtin_amdgcn_readfirstlane(s.prefix)};
}

// The key tiles that rows of the new tokens [i0, i1] of a sequence see: `sink_tiles` first ones and those from `sink_tiles + skip` on, `count`
// in all.  Tile u of them is tile u or u + skip of the sequence.  `first`: what none of the rows sees lies in front of it, but for a prefix and sinks.
struct Keys {
  int sink_tiles, skip, count;
};
static __device__ __forceinline__ Keys keys_of(const Seq& s, int i0, int i1, int causal, int window, int sinks, int first = 0) {
  const int before = s.len - s.n;  // tokens that were there (negative: queries that see nothing)
  const int end = max(causal ? min(s.len, before + i1 + 1) : s.len, s.prefix);
  Keys k{0, 0, 0};
  if (end <= 0) return k;
  const int tiles = (end + kKeyTile - 1) / kKeyTile;
  if (window > 0 || first > 0) {
    const int low = max(first, window > 0 ? before + i0 + 1 - window : 0);
    k.sink_tiles = (max(min(sinks, end), s.prefix) + kKeyTile - 1) / kKeyTile;
    k.skip = max(0, min(low / kKeyTile, tiles) - k.sink_tiles);
  }
  k.count = tiles - k.skip;
  return k;
}

// What a sequence brings to a launch: row tiles of few or of many rows, and the most key tiles that one of them sees.
template <bool MANY, int SC> static __device__ __forceinline__ void load_of(const AttendArgs& a, const Seq& s, int& tiles, int& keys) {
  constexpr int ROWS = MANY ? kManyRows : kFewRows;
  const int rows = s.n * a.group;
  tiles = (rows > a.few_most) == MANY ? (rows + ROWS - 1) / ROWS : 0;
  keys = keys_of(s, 0, s.n - 1, a.causal, a.window, a.sinks).count;
  if (a.window > 0) {  // a row tile sees no more than its own window, wherever that begins, and the first tokens
    const int most = (a.window + ROWS - 1 + kKeyTile - 1) / kKeyTile + 1 + (max(a.sinks, s.prefix) + kKeyTile - 1) / kKeyTile;
    keys = min(keys, most);
  }
  // Documents that lie one behind the other: what is in front of the first token's no other token sees.  (Where that is not so the work is dealt out
  // unevenly.  20 sequences of 3 to 24 K tokens, 40 new ones each in documents of 12, 16 heads x 64: 92 us dealt by their lengths, 28 so; 42 single tokens over 0.4
  // to 4.4 K in documents of 90, 32/16 heads x 128, 61 and 16.)
  if (SC != 0 && a.x.first && s.n > 0 && s.len > s.n) {
    const int from = min(clamped(a.x.first[s.start], 0, s.len), s.len - s.n);
    keys = min(keys, (s.len - from) / kKeyTile + 2 + (max(a.sinks, s.prefix) + kKeyTile - 1) / kKeyTile);
  }
  keys = max(keys, 1);  // rows that see nothing are written too
}

// Inclusive sums over the lanes of a wave: within rows of 16 lanes, then from row to row.
static __device__ __forceinline__ int wave_scan(int x) {
  auto plus = [&](auto ctrl, auto rows) { x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, true); };
  using all = std::integral_constant<int, 0xf>;
  plus(std::integral_constant<int, 0x111>{}, all{});  // row_shr:1
  plus(std::integral_constant<int, 0x112>{}, all{});
  plus(std::integral_constant<int, 0x114>{}, all{});
  plus(std::integral_constant<int, 0x118>{}, all{});
  plus(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // lane 15 of rows 0 and 2 to rows 1 and 3
  plus(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // lane 31 to rows 2 and 3
  return x;
}
static __device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
static __device__ __forceinline__ float wave_sum(float x) {
  auto plus = [&](auto ctrl, auto rows) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, true));
  };
  using all = std::integral_constant<int, 0xf>;
  plus(std::integral_constant<int, 0x111>{}, all{});
  plus(std::integral_constant<int, 0x112>{}, all{});
  plus(std::integral_constant<int, 0x114>{}, all{});
  plus(std::integral_constant<int, 0x118>{}, all{});
  plus(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  plus(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The least and the largest first key of the new tokens [i0, i1] of a sequence (a.x.first), of a whole wave.
struct Firsts {
  int least, most;
};
static __device__ __forceinline__ Firsts firsts_of_lanes(int least, int most) {
  auto meet = [&](auto ctrl, auto rows) {  // (as wave_scan; a lane without a partner meets itself)
    least = min(least, __builtin_amdgcn_update_dpp(least, least, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    most = max(most, __builtin_amdgcn_update_dpp(most, most, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using all = std::integral_constant<int, 0xf>;
  meet(std::integral_constant<int, 0x111>{}, all{});
  meet(std::integral_constant<int, 0x112>{}, all{});
  meet(std::integral_constant<int, 0x114>{}, all{});
  meet(std::integral_constant<int, 0x118>{}, all{});
  meet(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  meet(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return Firsts{__builtin_amdgcn_readlane(least, 63), __builtin_amdgcn_readlane(most, 63)};
}
static __device__ __forceinline__ Firsts firsts_of(const Scoring& x, const Seq& s, int i0, int i1) {
  if (!x.first) return Firsts{0, 0};
  int least = INT32_MAX, most = 0;
  for (int i = i0 + (int)(threadIdx.x & 63); i <= i1; i += 64) {
    const int f = clamped(x.first[s.start + i], 0, s.len);
    least = min(least, f);
    most = max(most, f);
  }
  return firsts_of_lanes(least, most);
}

// Many rows: the key tiles of a row tile are cut into even shares, so many that the whole launch makes about kManyWorkgroups workgroups,
// each of kManyLeast tiles at least.  (A chunk of 512 over 2 K, 8 heads, us with 8, 12, 16 and 32 tiles: 28, 31, 35, 45.)
struct Place {
  Seq s;
  int b;
  int tile, split, splits;  // row tile, which share of its key tiles of how many
  int slot;                 // where the part of the row tile's first share lies (splits > 1)
};
// The place-th share of a KV head; MERGE: the place-th row tile that was cut.  Every wave works it out for itself, a lane a sequence, so that
// there is no barrier.  False beyond the last.
template <bool MERGE, int SC> static __device__ __forceinline__ bool find_place(const AttendArgs& a, int place, Place& p) {
  const int lane = threadIdx.x & 63;
  float total = 0.f;
  for (int b0 = 0; a.many_cut && b0 < a.c.batch; b0 += 64) {
    float work = 0.f;
    if (b0 + lane < a.c.batch) {
      int tiles, keys;
      load_of<true, SC>(a, seq_of(a.c, b0 + lane, SC ? a.x.prefix : nullptr), tiles, keys);
      work = (float)tiles * (float)keys;
    }
    total += wave_sum(work);
  }
  const float share = fmaxf(total * a.kv_heads / kManyWorkgroups, (float)kManyLeast);
  int before = 0, slots_before = 0;
  for (int b0 = 0; b0 < a.c.batch; b0 += 64) {
    Seq s{0, 0, 0, 0};
    int tiles = 0, splits = 1;
    if (b0 + lane < a.c.batch) {
      int keys;
      s = seq_of(a.c, b0 + lane, SC ? a.x.prefix : nullptr);
      load_of<true, SC>(a, s, tiles, keys);
      splits = a.many_cut ? max(1, (int)ceilf(keys / share)) : 1;
      // Of a scored call no more shares than run at once, where there is that much to do, and none that leave a row tile less than kManySaved shorter: a part's
      // way through memory and the putting together cost as much.  (Us with shares as those of plain calls and so, 32 heads on 4 x 128: chunks of 147 to 315 tokens
      // in a window of 78 41 and 29, five sequences of some 1 K in documents of 50 49 and 25; prompts of 90 to 1000 tokens, 16 heads on 8, 56 and 50; four
      // chunks of some 300 over 500 to 900, 16 heads on 4, 37 and 43; a prompt of 700 31 and 31.)
      if (SC != 0 && share > (float)kManyLeast) splits = max(1, (int)(keys / share + 0.01f));
      if (SC != 0 && (!a.many_cut || keys - (keys + splits - 1) / splits < kManySaved)) splits = 1;
    }
    int b = b0 + lane;
    // Of a scored call of up to 64 sequences, those first whose shortest row tile sees most: rows of long contexts that start when all others are done
    // are waited for.  (Prompts of 4 K and 1.3 K beside 1 K over 4 K and single tokens, 16 heads x 128, slopes: 198 us in the sequences' order, and 184; two
    // chunks over 4 K, 16 heads on 4, 91 and 92, and 105 where every wave looks at 64 lanes in place of the sequences there are.)
    if constexpr (SC != 0) {
      if (a.c.batch <= 64 && a.c.batch > 1) {
        const int sees = tiles > 0 ? max(s.len - s.n, 0) : -1;
        int rank = max(lane - a.c.batch, 0);  // (lanes without a sequence stay behind)
        for (int l = 0; l < a.c.batch; ++l) {
          const int other = __builtin_amdgcn_readlane(sees, l);
          rank += other > sees || (other == sees && l < lane);
        }
        auto to_rank = [&](int x) { return __builtin_amdgcn_ds_permute(4 * rank, x); };
        s = Seq{to_rank(s.len), to_rank(s.start), to_rank(s.n), to_rank(s.prefix)};
        tiles = to_rank(tiles);
        splits = to_rank(splits);
        b = to_rank(b);
      }
    }
    const int shares = tiles * splits, slots = splits > 1 ? shares : 0, units = !MERGE ? shares : splits > 1 ? tiles : 0;
    const int upto = wave_scan(units), slots_upto = wave_scan(slots);
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(before + upto > place);
    if (beyond) {
      const int l = __builtin_ctzll(beyond);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      p.s = Seq{of(s.len), of(s.start), of(s.n), SC ? of(s.prefix) : 0};
      p.b = of(b);
      p.splits = of(splits);
      const int r = place - (before + of(upto) - of(units));
      const int first = slots_before + of(slots_upto) - of(slots);
      p.tile = MERGE ? r : r / p.splits;
      p.split = MERGE ? 0 : r - p.tile * p.splits;
      p.slot = first + p.tile * p.splits;
      p.tile = of(tiles) - 1 - p.tile;  // the rows that see most first
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    slots_before += __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return false;
}

// Parts go from workgroup to workgroup, which may sit on different XCDs with an L2 each: they are written through to and read from what all
// XCDs share.  With a release fence on the writers' side each writes back an L2: one token over 128 K, 16 heads 202 us with 256 workgroups,
// 248 with 1024; with an acquire fence on the readers' side each empties one: 48 single tokens over some 3 K 72 us instead of 70.
// Read eight bytes a lane, a row tile of 8 parts of 32 rows took 15 us to put together, 10 with a wave's bytes beside each other, 4 with 16 a lane.
static __device__ __forceinline__ void put_part(float* to, const f32x4& x) {
  // (the registers of a store of 16 bytes may not be written in the next cycle, which the compiler minds for stores of its own)
  asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(to), "v"(x) : "memory");
}
static __device__ __forceinline__ float2 get_stat(const float2* from) {
  return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
static __device__ __forceinline__ void put_stat(float2* to, const float2& x) {
  __hip_atomic_store((uint64_t*)to, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Byte offset of row `key` of a page's KV head from the start of the pool.
static __device__ __forceinline__ int64_t page_row(const Cache& c, int page, int head, int key) {
  return page * c.page_stride + head * c.head_stride + (int64_t)(key & ((1 << c.page_shift) - 1)) * c.token_stride;
}

// O = acc / l and the LSE of row r of a sequence's KV head, eight columns of it.
template <int DT>
static __device__ __forceinline__ void store_row(const AttendArgs& a, const Seq& s, int head, int r, int c8, float (&o)[8], float top, float l) {
  const int token = quotient(r, a.by_group), q_head = head * a.group + r - token * a.group;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] *= inv;
  char* to = a.out + (s.start + token) * a.o_ts + q_head * a.o_hs;
  if (a.out_fp32) {
    *(f32x4*)(to + c8 * 32) = f32x4{o[0], o[1], o[2], o[3]};
    *(f32x4*)(to + c8 * 32 + 16) = f32x4{o[4], o[5], o[6], o[7]};
  } else {
    Store8<DT>::st(to + c8 * 16, o);
  }
  if (c8 == 0) a.lse[(int64_t)q_head * a.c.tokens + s.start + token] = l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// The same for a 32-row block of a wave's accumulators (O^T: lane (n, h) has four columns of every eight of row n), as store_block
// stores it: rows [row0, r_last] of a sequence's KV head, 64 contiguous bytes of 16 rows at a time; NB 32-column blocks from db0 on.
template <int DT, int NB>
static __device__ __forceinline__ void store_rows(const AttendArgs& a, const Seq& s, int head, int row0, int r_last, const f32x16 (&acc)[NB], int db0,
                                                  float l, float ms) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
  auto at = [&](int r, char* base, int64_t ts, int64_t hs) {
    const int token = quotient(r, a.by_group);
    return base + (s.start + token) * ts + (head * a.group + r - token * a.group) * hs;
  };
  if (a.out_fp32) {
    if (row0 + n <= r_last) {
      char* to = at(row0 + n, a.out, a.o_ts, a.o_hs) + 128 * db0 + 16 * h;
#pragma unroll
      for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *(f32x4*)(to + 128 * db + 32 * q4) = f32x4{acc[db][4 * q4] * inv, acc[db][4 * q4 + 1] * inv, acc[db][4 * q4 + 2] * inv, acc[db][4 * q4 + 3] * inv};
    }
  } else {
    const int r = row0 + (lane & 15), c = 2 * ((lane >> 4) & 1) + (lane >> 5);  // row (and row + 16), 16-byte piece of the 64
    char* p0 = at(min(r, r_last), a.out, a.o_ts, a.o_hs) + 64 * db0 + 16 * c;
    char* p1 = at(min(r + 16, r_last), a.out, a.o_ts, a.o_hs) + 64 * db0 + 16 * c;
#pragma unroll
    for (int db = 0; db < NB; ++db) {
      u32x4 x, y;  // columns [0, 8) + 8 h, and 16 further on
      auto pack = [&](int e) {
        typedef typename Elem<DT>::type T;
        typedef T T2 __attribute__((ext_vector_type(2)));
        const T2 v = {(T)(acc[db][e] * inv), (T)(acc[db][e + 1] * inv)};
        return __builtin_bit_cast(unsigned, v);
      };
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x4& t = k == 0 ? x : y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto z = __builtin_amdgcn_permlane32_swap(pack(8 * k + 2 * i), pack(8 * k + 4 + 2 * i), false, false);
          t[i] = z[0];
          t[2 + i] = z[1];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto z = __builtin_amdgcn_permlane16_swap(x[e], y[e], false, false);
        x[e] = z[0];
        y[e] = z[1];
      }
      if (r <= r_last) *(u32x4*)(p0 + 64 * db) = x;
      if (r + 16 <= r_last) *(u32x4*)(p1 + 64 * db) = y;
    }
  }
  if (db0 == 0 && h == 0 && row0 + n <= r_last) {
    const int token = quotient(row0 + n, a.by_group), q_head = head * a.group + row0 + n - token * a.group;
    a.lse[(int64_t)q_head * a.c.tokens + s.start + token] = l == 0.f ? -INFINITY : (ms + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  }
}

// The pages of a wave's next 64 key tiles, a lane a tile: of its first 16 keys, of the 16 behind them; -1 where there is none.
struct HeldPages {
  int page0, page1;
  // key: the first of this lane's tile; `there`: whether it has one
  __device__ __forceinline__ void hold(const Cache& c, const int* table, int key, bool there) {
    page0 = page1 = -1;
    if (there) {
      const int e0 = key >> c.page_shift, e1 = (key + 16) >> c.page_shift;
      page0 = table[e0];
      page1 = e1 == e0 ? page0 : e1 < c.table_pages ? table[e1] : -1;
      if ((unsigned)page0 >= (unsigned)c.pages) page0 = -1;
      if ((unsigned)page1 >= (unsigned)c.pages) page1 = -1;
    }
  }
};
// 16 keys x D to LDS, 1 KB a piece: offsets of this lane's 16 bytes of each piece from the first key's row.  A load's own offset moves
// both ends, and the cache's rows may lie further apart than those in LDS: the difference is in the offsets.
template <int D, class Swizzle> static __device__ __forceinline__ void half_tile_offsets(int (&goff)[D / 32], int token_stride, Swizzle swizzle) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const int r = 512 / D * j + lane / (D / 8);
    goff[j] = r * token_stride - 1024 * j + (((lane % (D / 8)) ^ swizzle(r)) << 4);
  }
}
// Non-temporal: these rows are read once, and what all compute units have on the way at a time is as large as L2 (us with and without: 48
// sequences of some 4 K tokens, 16/4 heads 74.8, 84.4; one of 128 K, 16 heads 190.6, 198.9).
template <bool ONCE, int HALF> static __device__ __forceinline__ void load_half_tile(const char* base, unsigned dst, const int (&goff)[HALF]) {
#define RA_LOAD(hint)                                                                                                                             \
  do {                                                                                                                                            \
    if constexpr (HALF == 4)                                                                                                                      \
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %5" hint "\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024" hint      \
                   "\n\tglobal_load_lds_dwordx4 %3, %5 offset:2048" hint "\n\tglobal_load_lds_dwordx4 %4, %5 offset:%6" hint ::"s"(              \
                       __builtin_amdgcn_readfirstlane(dst)),                                                                                      \
                   "v"(goff[0]), "v"(goff[1]), "v"(goff[2 % HALF]), "v"(goff[3 % HALF]), "s"(base), "n"(3 << 10)                                  \
                   : "m0");                                                                                                                       \
    else                                                                                                                                          \
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %3" hint "\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024" hint ::"s"( \
                       __builtin_amdgcn_readfirstlane(dst)),                                                                                      \
                   "v"(goff[0]), "v"(goff[1 % HALF]), "s"(base)                                                                                   \
                   : "m0");                                                                                                                       \
  } while (0)
  if constexpr (ONCE) RA_LOAD(" nt");
  else RA_LOAD("");
#undef RA_LOAD
}

// The same with scores that are shaped; which: SC.
hipError_t launch_paged_scored(const AttendArgs& a, int sc, int dtype, int dim, int64_t many_places, int64_t cut_tiles, hipStream_t stream);

// A launch of kFewWorkgroups workgroups and `many_places` more for each KV head; a.many_cut: and one that puts together the row tiles
// whose keys were shared out, of which there are up to `cut_tiles`.
hipError_t launch_paged_attend(const AttendArgs& a, int dtype, int dim, int64_t many_places, int64_t cut_tiles, hipStream_t stream);

struct AppendArgs {
  Cache c;
  const char* k;
  const char* v;
  int64_t ts, hs;  // bytes between tokens, between heads
  float* scores;   // [pages, kv_heads, page] or NULL
  int kv_heads;
};
hipError_t launch_paged_append(const AppendArgs& a, int dim, hipStream_t stream);

struct WeightsArgs {
  Cache c;
  Scoring x;
  const char* q;
  const float* lse;  // [heads, tokens]
  float* scores;     // [pages, kv_heads, page]
  int64_t q_ts, q_hs;
  int kv_heads, group;
  Divisor by_group;
  float scale_log2;
  int causal, window, sinks;
  int few_most;  // as in AttendArgs
  int q_even;    // 32 rows are whole tokens, and lie within 2 GiB
  float* parts;  // many rows: sums of the parts of a block of keys, kManyKeys each
  int* arrived;  // ... and how many of them are there; 0 between launches
};
hipError_t launch_paged_weights(const WeightsArgs& a, int sc, int dtype, int dim, hipStream_t stream);

struct EvictArgs {
  Cache c;
  float* scores;         // [pages, kv_heads, page]
  const int* kept_table; // [batch, kept pages]
  int64_t kept_stride;
  int kept_pages;
  int budget, first, last;
  int present;     // tokens whose page is not there do not stay
  int* kept;       // [batch, kv_heads, budget]
  int* kept_lens;  // [batch]
  int kv_heads;
  void* workspace;
  size_t workspace_bytes;
};
hipError_t launch_paged_evict(const EvictArgs& a, int dim, hipStream_t stream);

}  // namespace paged
}  // namespace ringattn
