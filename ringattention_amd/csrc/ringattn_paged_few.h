// gfx950 (CDNA4): attention of few new tokens over a paged cache, the workgroup's program (ringattn_paged_attend.hip wraps it).
//
// 32 query rows (tokens x heads of a group) of one KV head of a sequence against a range of the key tiles that they see.  Eight waves
// take the range's 32-key tiles in turn, each with a softmax state of its own, as in ring_split_kernel: S^T = K Q^T and O^T += V^T P^T on
// 32x32x16 MFMAs, K and V HBM -> LDS -> fragments without a barrier, one buffer of each per wave; the states meet in LDS at the end.
//
// A row of few has nothing to reuse: every K and V row is read once from memory for the rows of a group, so that memory is what bounds
// it, and that wants every compute unit to read all the time.  So the key tiles of all row tiles of a launch are laid end to end and
// cut into as many equal runs as there are workgroups, whatever the lengths of the sequences: a workgroup goes through its run row
// tile by row tile.  A row tile that a run ends in is put together by the last of the workgroups that have a part of it, in the
// order of the parts: no second launch, and the same bits whoever is last.
#pragma once
#include "ringattn_paged.h"

namespace ringattn {
namespace paged {

// The row tiles of a launch laid end to end, as units of key tiles: of 64 sequences, a lane each.
struct Lanes {
  Seq s;
  int tiles, keys;  // row tiles, and units of each (an upper bound of what its rows see, the same for all of a sequence)
  int upto;         // units of all sequences up to this one
  int most = 0, fewest = INT32_MAX;  // key tiles that a row tile of any sequence sees
  float news = 0.f;                  // new tokens of this lane's sequences
  // round: to multiples of kFewLeast; else kFewSmall at least, or `fixed` of them
  __device__ __forceinline__ int add(const AttendArgs& a, int b0, int before, bool round, int fixed) {
    const int lane = threadIdx.x & 63;
    s = Seq{0, 0, 0};
    tiles = 0;
    keys = 1;
    if (b0 + lane < a.c.batch) {
      s = seq_of(a.c, b0 + lane);
      news += (float)s.n;
      load_of<false>(a, s, tiles, keys);
      if (tiles > 0) {
        most = max(most, keys);
        fewest = min(fewest, keys);
      }
      keys = round ? (keys + kFewLeast - 1) / kFewLeast * kFewLeast : max(keys, kFewSmall);
      keys = fixed > 0 ? fixed : ((keys - 1) >> a.few_shift) + 1;
    }
    upto = before + wave_scan(tiles * keys * a.kv_heads);
    return __builtin_amdgcn_readlane(upto, 63);
  }
};
// What lies at a place of theirs.
struct Piece {
  Seq s;
  int b, tile, head;
  int from, keys;   // unit of the row tile, of how many
  __device__ __forceinline__ bool find(const AttendArgs& a, const Lanes& x, int b0, int pos) {
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(x.upto > pos);
    if (beyond == 0) return false;
    const int l = __builtin_ctzll(beyond);
    auto of = [&](int y) { return __builtin_amdgcn_readlane(y, l); };
    s = Seq{of(x.s.len), of(x.s.start), of(x.s.n)};
    b = b0 + l;
    keys = of(x.keys);
    const int at = pos - (of(x.upto) - of(x.tiles) * keys * a.kv_heads), unit = at / keys;
    from = at - unit * keys;
    head = of(x.tiles) == 1 ? unit : unit / of(x.tiles);
    tile = unit - head * of(x.tiles);
    return true;
  }
};

// A part's row, eight columns of it: 16 bytes of every thread beside each other, twice.
template <int D> static __device__ __forceinline__ void put_row(const AttendArgs& a, int slot, int r, int c8, const float (&o)[8], float top, float l) {
  const int64_t prow = (int64_t)slot * kFewRows + r;
  float* to = a.few.o + prow * D + c8 * 4;
  put_part(to, f32x4{o[0], o[1], o[2], o[3]});
  put_part(to + D / 2, f32x4{o[4], o[5], o[6], o[7]});
  if (c8 == 0) put_stat(a.few.stat + prow, float2{top, l});
}

// The parts of a row tile, `count` rows of it, put together by all threads of the workgroup: a thread has eight columns of a row and
// every so-many-th of its parts, and those of a row meet in LDS.  slot(i): where part i lies; to: where their sum goes as one part, or -1: these
// are all of the row tile's.
template <int DT, int D, class Slot>
static __device__ __forceinline__ void merge_parts(const AttendArgs& a, const Seq& s, int head, int r0, int count, int parts, Slot slot, int to,
                                                   float (*sums)[10]) {
  constexpr int TPR = D / 8, GROUPS = 512 / TPR;
  int at_once = 1;  // rows at once; the groups of threads left share a row's parts
  while (at_once < count) at_once *= 2;
  const int sharers = min(GROUPS / at_once, 8);  // (more would meet longer than they fetch)
  const int g = threadIdx.x / TPR, c8 = threadIdx.x % TPR;
  const int sub = g / at_once, r = sub < sharers ? g % at_once : count;
  float top = -INFINITY, l = 0.f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  auto add = [&](float ref, float sum, const f32x4& x0, const f32x4& x1) {  // (a reference of -inf: nothing seen)
    const float t = fmaxf(top, ref), z = t == -INFINITY ? 0.f : t, keep = __builtin_amdgcn_exp2f(top - z), w = __builtin_amdgcn_exp2f(ref - z);
    l = ref == -INFINITY ? l : __builtin_fmaf(sum, w, l * keep);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = ref == -INFINITY ? o[e] : __builtin_fmaf(x0[e], w, o[e] * keep);
      o[4 + e] = ref == -INFINITY ? o[4 + e] : __builtin_fmaf(x1[e], w, o[4 + e] * keep);
    }
    top = t;
  };
  // reads past the caches (bit 4 of the cache policy), 16 bytes a lane: as a buffer, whose loads the compiler waits for itself
  const auto buffer = __builtin_amdgcn_make_buffer_rsrc(a.few.o, 0, kFewSlots * kFewRows * D * 4, 0x00027000);
  auto fetch = [&](int at) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer, at, 0, 16)); };
  if (r < count) {
    constexpr int kBatch = 4;  // parts on their way together
#pragma unroll 1
    for (int i = sub; i < parts; i += kBatch * sharers) {
      float2 st[kBatch];
      f32x4 x0[kBatch], x1[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int prow = slot(min(i + j * sharers, parts - 1)) * kFewRows + r, at = prow * (D * 4) + c8 * 16;
        st[j] = get_stat(a.few.stat + prow);
        x0[j] = fetch(at);
        x1[j] = fetch(at + D * 2);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) add(i + j * sharers < parts ? st[j].x : -INFINITY, st[j].y, x0[j], x1[j]);
    }
  }
  if (sharers > 1) {
    float* mine = sums[threadIdx.x];
    mine[0] = top;
    mine[1] = l;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[2 + e] = o[e];
    __syncthreads();
    if (sub == 0) {
#pragma unroll 1
      for (int i = 1; i < sharers; ++i) {
        const float* x = sums[threadIdx.x + i * at_once * TPR];
        add(x[0], x[1], f32x4{x[2], x[3], x[4], x[5]}, f32x4{x[6], x[7], x[8], x[9]});
      }
    }
  }
  if (sub != 0 || r >= count) return;
  if (to < 0) {
    store_row<DT>(a, s, head, r0 + r, c8, o, top, l);
  } else {  // (into a slot that this thread alone, or one of its row's, has read)
    put_row<D>(a, to, r, c8, o, top, l);
  }
}

template <int D> constexpr int kFewWaveLds = 2 * kKeyTile * D * 2;  // a K and a V tile; at the end the wave's acc-O
// A part that a run leaves of a row tile: which rows, and how many parts there are from which run on.
struct Left {
  Seq s;
  int head, r0, count, first_run, parts, last;
};
template <int D> constexpr int kFewLds = 8 * kFewWaveLds<D> + 8 * kFewRows * (int)sizeof(float2) + 2 * (int)sizeof(Left) + 16 * (int)sizeof(int);

template <int DT, int D> static __device__ __forceinline__ void few_rows(const AttendArgs& a, unsigned char* smem, int block) {
  using E = Elem<DT>;
  constexpr int WAVES = 8, BM = kFewRows, BN = kKeyTile;
  constexpr int ROWB = D * 2, TILE = BN * ROWB;
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int PIECES = TILE / 1024;     // 1 KB wave-loads per tile
  constexpr int HALF = PIECES / 2;        // ... per 16 keys, which always lie in one page
  constexpr int WREG = kFewWaveLds<D>;
  static_assert(WREG >= BM * D * 4, "acc-O of a wave as fp32 takes the place of its tiles");
  static_assert(WAVES * WREG >= 512 * 10 * 4, "sums of merge_parts");
  float2 (*stat)[BM] = (float2 (*)[BM])(smem + WAVES * WREG);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;

  // The runs: `each` units of all of them.  Every wave works out for itself where its run lies, without a barrier; up to 64 sequences stay
  // in its registers.
  Lanes lanes;
  // Where runs of kFewLeast key tiles suffice for all, every row tile begins a run.  Elsewhere a row tile, whatever it sees, costs its
  // beginning and end, some 5 us, and the parts' way through memory where a run ends inside it: it counts as kFewSmall key tiles at
  // least, and where none sees more, runs are of whole row tiles.  (Us with neither, and with 16 and 32 for kFewSmall: 113 sequences of one
  // token, 4 heads 79, 23, 10; 40 of 700, 8 KV heads -, 35, 30; 48 of some 3 K, 4 KV heads 75, 73, 70.  With 32 for kFewLeast one of 4 K, 8 KV
  // heads takes 15 instead of 14, and one of 16 K has half as many workgroups.)
  const int least = max(1, kFewLeast >> a.few_shift), small = max(1, kFewSmall >> a.few_shift);  // units
  int total = 0;
  for (int b0 = 0; b0 < a.c.batch; b0 += 64) total = lanes.add(a, b0, total, true, 0);
  // Starts that go down and up again have sequences share the call's tokens, and a.few_shift lets 32 bits suffice for sequences that do not: with
  // as many new tokens in all as the call has, 2^30.  Where they have more than a few shared ones, nothing is done for those of few rows.
  if (wave_sum(lanes.news) > 1.75f * a.c.tokens) return;
  const bool round = total <= kFewWorkgroups * least, all_small = __builtin_amdgcn_ballot_w64(lanes.most > kFewSmall) == 0;
  const bool some_small = !round && __builtin_amdgcn_ballot_w64(lanes.fewest <= kFewSmall) != 0;
  if (!round) {
    total = 0;
    for (int b0 = 0; b0 < a.c.batch; b0 += 64) total = lanes.add(a, b0, total, false, 0);
  }
  int each = round ? least : max((total + kFewWorkgroups - 1) / kFewWorkgroups, least);
  if (!round && all_small) each = (each + small - 1) / small * small;
  // Row tiles that all see as much -- one sequence, or several as long as each other -- are cut into as many runs each, where that takes no less
  // than 7/8 of the workgroups, so that no run ends inside one.  (Us with and without, 32 heads on 8: 16 tokens over 32800 34 and 54, over 10000 21 and 34; 16 single
  // tokens over 4 K, 4 KV heads 30 and 35; one over 50 K, 16 heads 77 and 84.)
  int fixed = 0;
  if (!round && !all_small) {
    const uint64_t have = __builtin_amdgcn_ballot_w64(lanes.most > 0);
    const int same = __builtin_amdgcn_readlane(lanes.most, __builtin_ctzll(have));
    if (__builtin_amdgcn_ballot_w64(lanes.most > 0 && (lanes.most != same || lanes.fewest != same)) == 0) {
      const int units = ((same - 1) >> a.few_shift) + 1, row_tiles = total / units, runs_each = kFewWorkgroups / max(row_tiles, 1);
      if (row_tiles * runs_each >= kFewWorkgroups * 7 / 8) {
        each = (units + runs_each - 1) / runs_each;
        fixed = each * runs_each;
        total = row_tiles * fixed;
        lanes.upto = lanes.upto / units * fixed;
        lanes.keys = fixed;
      }
    }
  }
  // Runs beside each other on one XCD, an eighth of them each: row tiles of a sequence's KV head, which read the same keys, find them in its L2.
  const int runs = round ? total >> __builtin_ctz(least) : (total - 1) / each + 1, of_xcd = (runs + 7) / 8, w = (block & 7) * of_xcd + (block >> 3);
  if (block >> 3 >= of_xcd || w >= runs) return;
  const int end = min((int64_t)total, (int64_t)(w + 1) * each);
  // The parts that this run leaves: of a row tile that began before it, and of one that goes on behind it.  They are counted when the
  // run is through, and not each on its own, which would keep the workgroup waiting for its stores (some 8 us a part).
  Left* left = (Left*)(smem + WAVES * WREG + WAVES * BM * sizeof(float2));
  if (tid < 2) left[tid].parts = 0;

  int (*counts)[WAVES] = (int (*)[WAVES])((unsigned char*)left + 2 * sizeof(Left));
  for (int pos = w * each, turn = 0; pos < end; turn ^= 1) {
    auto find = [&](Piece& p, int at) {
      if (a.c.batch <= 64) {
        p.find(a, lanes, 0, at);
      } else {
        for (int b0 = 0, before = 0; b0 < a.c.batch; b0 += 64) {
          before = lanes.add(a, b0, before, round, fixed);
          if (p.find(a, lanes, b0, at)) break;
        }
      }
    };
    auto keys_at = [&](const Piece& p) {
      const int first = p.tile * BM, last = min(first + BM, p.s.n * a.group) - 1;
      return keys_of(p.s, quotient(first, a.by_group), quotient(last, a.by_group), a.causal, a.window, a.sinks);
    };
    // Where some of the next eight row tiles see little, each is a wave's own: they begin and end beside each other, and do not meet.  Against eight
    // waves a row tile one after the other, that is `most` tiles in a wave instead of `in_row` beginnings and ends.  (Us alone and not: 94
    // sequences of some six tokens, 8 KV heads 10 and 30; 81 of some 1 K and a window of 48, 32 heads, some with 40 new tokens 63 and
    // 130; 110 of some 90 tokens, 4 heads 21 and 28.)
    Piece p;
    const int mine = pos + wave * small;  // (where this wave's begins if those before it are as small)
    bool alone = false;
    int in_row = 0;
    if (some_small) {
      int count = -1;
      if (mine + small <= end) {
        find(p, mine);
        if (p.from == 0 && p.keys == small) count = keys_at(p).count;
      }
      counts[turn][wave] = count;
      __syncthreads();
      int most = 0;
      bool on = true;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const int c = __builtin_amdgcn_readfirstlane(counts[turn][i]);
        on = on && c >= 0;
        if (on) {
          ++in_row;
          most = max(most, c);
        }
      }
      alone = most <= 4 * (in_row - 1);
    }
    if (!alone) find(p, pos);
    else if (wave >= in_row) {
      pos += in_row * small;
      continue;
    }
    const int begin = alone ? mine : pos, upto = min(p.keys, p.from + (end - begin)), unit_begin = begin - p.from;
    pos += alone ? in_row * small : upto - p.from;
    const int rows = p.s.n * a.group, head = p.head;
    const int r0 = p.tile * BM, r_last = min(r0 + BM, rows) - 1;
    const int i0 = quotient(r0, a.by_group), i1 = quotient(r_last, a.by_group);
    const Keys keys = keys_at(p);
    auto tile_at_unit = [&](int u) { return p.keys == keys.count || u == 0 ? u : u == p.keys ? keys.count : (int)((int64_t)u * keys.count / p.keys); };
    const int u_begin = tile_at_unit(p.from), u_end = tile_at_unit(upto);

    // this lane's row: its token, its head, its position; rows beyond the range read the last valid one
    const int row = min(r0 + n, r_last), token = quotient(row, a.by_group), q_head = head * a.group + row - token * a.group;
    const int before = p.s.len - p.s.n;
    const int lim = a.causal ? min(p.s.len, before + token + 1) : p.s.len;           // keys below it are visible ...
    const int low = a.window > 0 ? before + token - a.window : -1;                   // ... if they are above this one, or sinks
    // of all rows of the tile
    const int lim_all = a.causal ? min(p.s.len, before + i0 + 1) : p.s.len, low_any = a.window > 0 ? before + i1 - a.window : -1;

    s16x8 qf[KS];
    {
      const char* qrow = a.q + (p.s.start + token) * a.q_ts + q_head * a.q_hs + h * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const s16x8*)(qrow + ks * 32);
    }

    unsigned char* my = smem + wave * WREG;
    const unsigned my_lds = lds_offset(smem) + wave * WREG;
    const int koff0 = n * ROWB + ((h ^ k_swizzle<D>(n)) << 4);
    auto koff = [&](int ks) {  // the number of the slice in bits that are free: one register, not eight (which would be kept elsewhere)
      int o = koff0;
      if (ks > 0) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(o) : "n"(32 * ks), "v"(koff0));
      return o;
    };
    int voff0;
    {
      const int s = lane & 15, g1 = (lane >> 4) & 1;
      const int row8 = 4 * h + (s >> 2), c = 2 * g1 + ((s & 3) >> 1);
      voff0 = TILE + row8 * ROWB + ((c ^ v_swizzle<D>(row8)) << 4) + ((s & 1) << 3);
    }
    auto voff = [&](int db) {
      int o = voff0;
      if (db > 0) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(o) : "n"(64 * db), "v"(voff0));
      return o;
    };
    int goff_k[HALF], goff_v[HALF];
    half_tile_offsets<D>(goff_k, a.c.token_stride, [](int r) { return k_swizzle<D>(r); });
    half_tile_offsets<D>(goff_v, a.c.token_stride, [](int r) { return v_swizzle<D>(r); });

    // ---- the tiles of this wave: u_begin + wave, + 8, ..., or all
    const int stride_log = alone ? 0 : 3;
    static_assert(WAVES == 8, "");
    const int* table = a.c.table + (int64_t)p.b * a.c.table_stride;
    auto real_tile = [&](int u) { return u < keys.sink_tiles ? u : u + keys.skip; };
    HeldPages held;
    int first_held = 0;
    auto hold_pages = [&](int u) {
      first_held = u;
      const int lanes_tile = u + (lane << stride_log);
      held.hold(a.c, table, real_tile(lanes_tile) * BN, lanes_tile < u_end);
    };
    struct Tile {
      int key;             // its first key
      int gone;            // bit 0, 1: the page of its first, second 16 keys is not there (page 0 is read in its place, and hidden)
      int64_t at0, at1;
    };
    auto tile_at = [&](int u) {
      if ((u - first_held) >> stride_log >= 64) hold_pages(u);
      Tile x;
      x.key = real_tile(u) * BN;
      const int l = (u - first_held) >> stride_log;
      const int e0 = __builtin_amdgcn_readlane(held.page0, l), e1 = __builtin_amdgcn_readlane(held.page1, l);
      x.gone = (e0 < 0 ? 1 : 0) | (e1 < 0 ? 2 : 0);
      x.at0 = page_row(a.c, max(e0, 0), head, x.key);
      x.at1 = page_row(a.c, max(e1, 0), head, x.key + 16);
      return x;
    };
    auto issue = [&](const char* pool, const Tile& x, unsigned dst, const int (&goff)[HALF]) {
      if (rows <= BM) {
        load_half_tile<true>(pool + x.at0, dst, goff);
        load_half_tile<true>(pool + x.at1, dst + TILE / 2, goff);
      } else {  // other row tiles read them too
        load_half_tile<false>(pool + x.at0, dst, goff);
        load_half_tile<false>(pool + x.at1, dst + TILE / 2, goff);
      }
    };
    auto issue_k = [&](const Tile& x) { issue(a.c.k, x, my_lds, goff_k); };
    auto issue_v = [&](const Tile& x) { issue(a.c.v, x, my_lds + TILE, goff_v); };

    float m = -INFINITY, ms = kNoReference, ls[4] = {0.f, 0.f, 0.f, 0.f};
    f32x16 oacc[DB], sacc;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
    s16x8 pf[2];
    float sums[4];
    // P = exp2(S k2 - m k2); the sums from the unrounded values, the operands of the next product rounded to the storage type: 2^-9 (bf16)
    // or 2^-12 (fp16) of a probability on average, no more than the output's own rounding
    auto exponentials = [&]() {
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) {
        typename E::vec8 pv;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[8 * t2 + e], a.scale_log2, -ms));
          sums[e & 3] = t2 == 0 && e < 4 ? x : sums[e & 3] + x;
          pv[e] = (typename E::type)x;
        }
        pf[t2] = __builtin_bit_cast(s16x8, pv);
      }
    };
    auto move_reference = [&]() {
      float m0 = m, m1 = m;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        m0 = fmaxf(fmaxf(m0, sacc[e]), sacc[e + 1]);
        m1 = fmaxf(fmaxf(m1, sacc[e + 2]), sacc[e + 3]);
      }
      m = cross_half_max(fmaxf(m0, m1));
      const float cs = (m == -INFINITY) ? kNoReference : m * a.scale_log2;
      const float alpha = __builtin_amdgcn_exp2f(ms - cs);
#pragma unroll
      for (int i = 0; i < 4; ++i) ls[i] *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      ms = cs;
    };
    auto hidden = [&](const Tile& x, int e, int hh) {  // of accumulator e of a lane of half hh: is its key hidden from this lane's row?
      const int key = x.key + 8 * (e >> 2) + (e & 3) + 4 * hh;
      return bool((key >= lim) | ((key <= low) & (key >= a.sinks)) | (x.gone >> (e >> 3) & 1));  // (no branches)
    };

    int u = u_begin + (alone ? 0 : wave);
    bool more = u < u_end;
    Tile cur{}, nxt{};
    if (more) {
      hold_pages(u);
      cur = tile_at(u);
      issue_k(cur);
      issue_v(cur);
    }
    __builtin_amdgcn_s_waitcnt(0);  // retire the Q loads with a wait the compiler can see (and the first tiles)
    for (int pass = 1; more; pass = 0) {  // pass: 1 while there is no reference to take exponentials against
      u += 1 << stride_log;
      more = u < u_end;
      if (more) nxt = tile_at(u);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");  // K is in, V may still be on its way
      {
        s16x8 kfr[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kfr[ks] = *(const s16x8*)(my + koff(ks));
        // the fragments are in registers: the K buffer takes the next tile
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (more) issue_k(nxt);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) sacc = E::mma(kfr[ks], qf[ks], sacc);
      }
      const bool masked = cur.key + BN > lim_all || (cur.key <= low_any && cur.key + BN > a.sinks) || cur.gone;
      if (masked) {
        asm volatile("");  // (a branch, not sixteen selections in every tile)
#pragma unroll
        for (int e = 0; e < 16; ++e) sacc[e] = hidden(cur, e, h) ? -INFINITY : sacc[e];
      }
      // exponentials against the reference as it stands; the row maximum is only looked at when a sum of four of them is above
      // 2^14 (or not a number)
#pragma unroll 1
      for (;; pass = 1) {
        if (pass) move_reference();
        exponentials();
        const bool large = !(fmaxf(fmaxf(sums[0], sums[1]), fmaxf(sums[2], sums[3])) <= 16384.f);
        if (pass || __builtin_amdgcn_ballot_w64(large) == 0) break;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) ls[i] += sums[i];
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PIECES) : "memory");  // V is in
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      // A hidden key's probability is 0, and 0 times an infinity or a NaN is not: where a masked tile's V holds such a value, the
      // product is taken key by key, over the visible ones.
      bool odd = false;
      if (masked) {
        unsigned top = 0;
#pragma unroll 4
        for (int i = 0; i < TILE / 1024; ++i) {
          typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
          const u32x4 x = *(const u32x4*)(my + TILE + 1024 * i + 16 * lane);
          constexpr unsigned kExp = DT == 0 ? 0x7c007c00u : 0x7f807f80u, kOne = DT == 0 ? 0x04000400u : 0x00800080u;
#pragma unroll
          for (int e = 0; e < 4; ++e) top |= (x[e] & kExp) + kOne;  // an exponent of ones carries into the sign's place
        }
        odd = __builtin_amdgcn_ballot_w64((top & 0x80008000u) != 0) != 0;
      }
      if (odd) {
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
          float mine = 0.f;
#pragma unroll
          for (int f = 0; f < 16; ++f) {
            const float x = (float)__builtin_bit_cast(typename E::vec8, pf[f >> 3])[f & 7];
            mine = e == f ? x : mine;
          }
          float of_lower = mine, of_upper = mine;
          swap_halves(of_lower, of_upper);
#pragma unroll 1
          for (int hh = 0; hh < 2; ++hh) {
            if (hidden(cur, e, hh)) continue;
            const float w = hh ? of_upper : of_lower;
            const int key = 8 * (e >> 2) + (e & 3) + 4 * hh;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                const typename E::vec4 x = *(const typename E::vec4*)(my + TILE + key * ROWB + (((4 * db + q4) ^ v_swizzle<D>(key)) << 4) + 8 * h);
#pragma unroll
                for (int i = 0; i < 4; ++i) oacc[db][4 * q4 + i] = __builtin_fmaf(w, (float)x[i], oacc[db][4 * q4 + i]);
              }
          }
        }
      } else {
        constexpr int AHEAD = 2;  // fragments read ahead of the MFMA that consumes one
        s16x8 vfr[2 * DB];
        auto read_v = [&](int f) {
          if (f >= 2 * DB) return;
          const unsigned char* vrow = my + 16 * (f / DB) * ROWB + voff(f % DB);
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vrow));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vrow + 8 * ROWB));
          vfr[f] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
#pragma unroll
        for (int f = 0; f < AHEAD; ++f) read_v(f);
#pragma unroll
        for (int f = 0; f < 2 * DB; ++f) {
          read_v(f + AHEAD);
          __builtin_amdgcn_sched_barrier(0);
          oacc[f % DB] = E::mma(vfr[f], pf[f / DB], oacc[f % DB]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) issue_v(nxt);
      cur = nxt;
    }

    if (alone) {
      store_rows<DT, DB>(a, p.s, head, r0, r_last, oacc, 0, cross_half_sum((ls[0] + ls[1]) + (ls[2] + ls[3])), ms);
      continue;
    }
    // This wave's state where the workgroup can read it: acc-O as fp32 over its own tiles, 16-byte chunk c of row n at chunk c ^ n.
    {
      const float l = cross_half_sum((ls[0] + ls[1]) + (ls[2] + ls[3]));
      if (h == 0) stat[wave][n] = float2{l == 0.f ? -INFINITY : ms, l};  // (0: nothing seen; a NaN stays one)
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          f32x4 val;
#pragma unroll
          for (int e = 0; e < 4; ++e) val[e] = oacc[db][4 * q4 + e];
          const int c = 8 * db + 2 * q4 + h;
          *(f32x4*)(my + n * (D * 4) + ((c ^ (n & (D / 4 - 1))) << 4)) = val;
        }
    }
    __syncthreads();
    constexpr int TPR = D / 8;  // threads of a row
    const int orow = tid / TPR, c8 = tid % TPR;
    const bool whole = p.from == 0 && upto == p.keys;
    const int first_run = unit_begin / each, slot = 2 * w + (w == first_run ? 1 : 0);
    if (orow <= r_last - r0) {
      float top = -INFINITY, l = 0.f, o[8];
#pragma unroll
      for (int i = 0; i < WAVES; ++i) top = fmaxf(top, stat[i][orow].x);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float2 st = stat[i][orow];
        const unsigned char* src = smem + i * WREG + orow * (D * 4);
        const f32x4 x0 = *(const f32x4*)(src + (((2 * c8) ^ (orow & (D / 4 - 1))) << 4));
        const f32x4 x1 = *(const f32x4*)(src + (((2 * c8 + 1) ^ (orow & (D / 4 - 1))) << 4));
        const float f = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - top);
        l = __builtin_fmaf(st.y, f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = __builtin_fmaf(x0[e], f, o[e]);
          o[4 + e] = __builtin_fmaf(x1[e], f, o[4 + e]);
        }
      }
      if (whole) {
        store_row<DT>(a, p.s, head, r0 + orow, c8, o, top, l);
      } else {
        put_row<D>(a, slot, orow, c8, o, top, l);
      }
    }
    if (!whole) {
      const int parts = (unit_begin + p.keys - 1) / each - first_run + 1;
      if (tid == 0) left[w == first_run ? 1 : 0] = Left{p.s, head, r0, r_last + 1 - r0, first_run, parts, 0};
    }
    __syncthreads();  // the next row tile's tiles and states go where these were
  }
  if (__builtin_amdgcn_readfirstlane(left[0].parts + left[1].parts) == 0) return;
  // Every wave waits for its own stores to be where all XCDs see them, the barrier for every wave, and only then the parts are counted; the
  // loads of one that finds itself the last are issued behind the barrier that follows its count.
  auto settle = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a barrier alone does not wait for stores)
    __syncthreads();
  };
  auto of = [&](int y) { return __builtin_amdgcn_readfirstlane(y); };
  auto count = [&](int* arrived, int parts) {  // whether this is the last of them
    const bool last = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    if (last) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
    return last;
  };
  settle();
  // Of more than kFewMerge parts, as many at a time become one first, by the last workgroup of theirs, and those the row tile: one that fetches
  // them all has long waits one after the other.  (One token, 128 K cached, one KV head, 16 heads: 93 us by one, 38 by 8, 16 or 32 at a
  // time; 32 heads 160 and 49.  16 KV heads have 16 parts each and do not come here.)
  if (tid < 2 && left[tid].parts > 0) {
    const int parts = left[tid].parts, first = left[tid].first_run, at = (w - first) & ~(kFewMerge - 1), some = min(kFewMerge, parts - at);
    // (one alone is not counted: its counter is that of the first ones of the row tile that begins in this run)
    if (parts <= kFewMerge) left[tid].last = count(a.few.arrived + first, parts);
    else left[tid].last = some == 1 || count(a.few.arrived + kFewWorkgroups + first + at, some);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const int parts = of(left[i].parts), first = of(left[i].first_run);
    if (parts == 0 || of(left[i].last) == 0) continue;
    const Seq s = uniform(left[i].s);
    const int head = of(left[i].head), r0 = of(left[i].r0), rows = of(left[i].count), at = (w - first) & ~(kFewMerge - 1);
    auto slot = [&](int k) { return 2 * (first + k) + (k == 0 ? 1 : 0); };
    // (one piece of code for both steps: it is fetched as it is first run, and that takes longer than what it does)
#pragma unroll 1
    for (int step = parts > kFewMerge ? kFewMerge : 1; step > 0;) {
      const bool whole = step == 1 && parts <= kFewMerge, group = step == kFewMerge;
      const int from = group ? at : 0, by = whole || group ? 1 : kFewMerge;
      const int n_parts = group ? min(kFewMerge, parts - at) : whole ? parts : (parts + kFewMerge - 1) / kFewMerge;
      merge_parts<DT, D>(a, s, head, r0, rows, n_parts, [&](int k) { return slot(from + k * by); }, group ? slot(at) : -1, (float (*)[10])smem);
      step = 0;
      if (group) {
        settle();
        if (tid == 0) left[i].last = count(a.few.arrived + first, (parts + kFewMerge - 1) / kFewMerge);
        __syncthreads();
        step = of(left[i].last);
      }
    }
    __syncthreads();
  }
}

}  // namespace paged
}  // namespace ringattn
