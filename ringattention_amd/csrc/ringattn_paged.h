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
constexpr int kManyWorkgroups = 256, kManyLeast = 8, kMergeSharers = 4;  // see find_place, merge_many
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

struct AttendArgs {
  Cache c;
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
};
static __device__ __forceinline__ int clamped(int x, int lo, int hi) { return min(max(x, lo), hi); }
// Lengths are data: whatever they hold, nothing outside the tensors is touched.  (A sequence's own are held to its table and to the call's tokens
// here; few_rows looks at what starts that do not ascend make of them all together.)
static __device__ __forceinline__ Seq seq_of(const Cache& c, int b) {
  Seq s;
  s.len = clamped(c.lens[b], 0, c.table_pages << c.page_shift);
  s.start = clamped(c.starts[b], 0, c.tokens);
  s.n = clamped(c.starts[b + 1], s.start, c.tokens) - s.start;
  return s;
}

static __device__ __forceinline__ Seq uniform(const Seq& s) {
  return Seq{__builtin_amdgcn_readfirstlane(s.len), __builtin_amdgcn_readfirstlane(s.start), __builtin_amdgcn_readfirstlane(s.n)};
}

// The key tiles that rows of the new tokens [i0, i1] of a sequence see: `sink_tiles` first ones and those from `sink_tiles + skip` on, `count`
// in all.  Tile u of them is tile u or u + skip of the sequence.
struct Keys {
  int sink_tiles, skip, count;
};
static __device__ __forceinline__ Keys keys_of(const Seq& s, int i0, int i1, int causal, int window, int sinks) {
  const int before = s.len - s.n;  // tokens that were there (negative: queries that see nothing)
  const int end = causal ? min(s.len, before + i1 + 1) : s.len;
  Keys k{0, 0, 0};
  if (end <= 0) return k;
  const int tiles = (end + kKeyTile - 1) / kKeyTile;
  if (window > 0) {
    const int low = max(0, before + i0 + 1 - window);
    k.sink_tiles = (min(sinks, end) + kKeyTile - 1) / kKeyTile;
    k.skip = max(0, min(low / kKeyTile, tiles) - k.sink_tiles);
  }
  k.count = tiles - k.skip;
  return k;
}

// What a sequence brings to a launch: row tiles of few or of many rows, and the most key tiles that one of them sees.
template <bool MANY> static __device__ __forceinline__ void load_of(const AttendArgs& a, const Seq& s, int& tiles, int& keys) {
  constexpr int ROWS = MANY ? kManyRows : kFewRows;
  const int rows = s.n * a.group;
  tiles = (rows > a.few_most) == MANY ? (rows + ROWS - 1) / ROWS : 0;
  keys = keys_of(s, 0, s.n - 1, a.causal, a.window, a.sinks).count;
  if (a.window > 0) {  // a row tile sees no more than its own window, wherever that begins, and the first tokens
    const int most = (a.window + ROWS - 1 + kKeyTile - 1) / kKeyTile + 1 + (a.sinks + kKeyTile - 1) / kKeyTile;
    keys = min(keys, most);
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
template <bool MERGE> static __device__ __forceinline__ bool find_place(const AttendArgs& a, int place, Place& p) {
  const int lane = threadIdx.x & 63;
  float total = 0.f;
  for (int b0 = 0; a.many_cut && b0 < a.c.batch; b0 += 64) {
    float work = 0.f;
    if (b0 + lane < a.c.batch) {
      int tiles, keys;
      load_of<true>(a, seq_of(a.c, b0 + lane), tiles, keys);
      work = (float)tiles * (float)keys;
    }
    total += wave_sum(work);
  }
  const float share = fmaxf(total * a.kv_heads / kManyWorkgroups, (float)kManyLeast);
  int before = 0, slots_before = 0;
  for (int b0 = 0; b0 < a.c.batch; b0 += 64) {
    Seq s{0, 0, 0};
    int tiles = 0, splits = 1;
    if (b0 + lane < a.c.batch) {
      int keys;
      s = seq_of(a.c, b0 + lane);
      load_of<true>(a, s, tiles, keys);
      splits = a.many_cut ? max(1, (int)ceilf(keys / share)) : 1;
    }
    const int shares = tiles * splits, slots = splits > 1 ? shares : 0, units = !MERGE ? shares : splits > 1 ? tiles : 0;
    const int upto = wave_scan(units), slots_upto = wave_scan(slots);
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(before + upto > place);
    if (beyond) {
      const int l = __builtin_ctzll(beyond);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      p.s = Seq{of(s.len), of(s.start), of(s.n)};
      p.b = b0 + l;
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
hipError_t launch_paged_weights(const WeightsArgs& a, int dtype, int dim, hipStream_t stream);

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
