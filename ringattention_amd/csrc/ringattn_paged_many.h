// gfx950 (CDNA4): attention of many new tokens over a paged cache, the workgroup's program (ringattn_paged_attend.hip wraps it).
//
// 256 query rows (tokens x heads of a group) of one KV head of a sequence and a share of the key tiles that they see; eight waves of 32
// rows, S^T = K Q^T and O^T += V^T P^T on 32x32x16 MFMAs, K and V HBM -> LDS in 32-key tiles through two rings of four, one barrier per
// two tiles.  As in ring_walk_kernel the two waves of a SIMD take turns: while one has its products the other has its softmax.
//
// What the pages add: a wave's 1 KB of a tile lies in one page, whose number a lane looked up for it 64 tiles at a time, and a tile's
// place is a product more; all rows of a page are memory of the pool, so the last tile of a sequence is read whole and masked.
#pragma once
#include "ringattn_paged.h"

namespace ringattn {
namespace paged {

template <int D> constexpr int kManyLds = 8 * kKeyTile * D * 2 + 16;

template <int DT, int D> static __device__ __forceinline__ void many_rows(const AttendArgs& a, unsigned char* smem, int block) {
  using E = Elem<DT>;
  constexpr int WAVES = 8, BM = kManyRows, BN = kKeyTile, NBUF = 4;
  constexpr int CPR = D / 8, ROWB = D * 2, TILE = BN * ROWB, KS = D / 16, DB = D / 32;
  constexpr int PIECES = TILE / 1024;  // 1 KB wave-loads per tile: 8 at d = 128, 4 at d = 64
  constexpr float kLazyLog2 = 8.f;
  static_assert(BM == 32 * WAVES, "one 32-row block per wave");
  static_assert(PIECES == WAVES || 2 * PIECES == WAVES, "a tile is loaded by all waves, or K and V by half of them each");

  const unsigned smem_base = lds_offset(smem);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;

  Place p;
  const int unit = quotient(block, a.by_kv_heads);
  const int head = block - unit * a.kv_heads;
  if (!find_place<false>(a, unit, p)) return;
  const int rows = p.s.n * a.group;
  const int r0 = p.tile * BM, r_last = min(r0 + BM, rows) - 1;
  const Keys keys = keys_of(p.s, quotient(r0, a.by_group), quotient(r_last, a.by_group), a.causal, a.window, a.sinks);
  const int u_begin = (int)((int64_t)p.split * keys.count / p.splits);
  const int n_tiles = (int)((int64_t)(p.split + 1) * keys.count / p.splits) - u_begin;  // of this share: tile t is tile u_begin + t

  // this lane's row; rows beyond the range read the last valid one
  const int row = min(r0 + 32 * wave + n, r_last), token = quotient(row, a.by_group), q_head = head * a.group + row - token * a.group;
  const int before = p.s.len - p.s.n;
  // What the masks and other seldom taken paths are worked out from: the compiler would keep all of it in registers through every tile.
  auto fresh = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  auto first_key = [&](int t) { return (u_begin + t < keys.sink_tiles ? u_begin + t : u_begin + t + keys.skip) * BN; };
  auto tile_of = [&](int real) { return (real < keys.sink_tiles ? real : max(keys.sink_tiles, real - keys.skip)) - u_begin; };
  // tiles that may need a mask: from `up` on, and below `low`; of this wave's rows, and of all rows of the workgroup
  struct Clear {
    int up, low;
  };
  auto clear_of = [&](int first, int last) {
    const int i0 = quotient(min(first, r_last), a.by_group), i1 = quotient(min(last, r_last), a.by_group);
    Clear x;
    x.up = __builtin_amdgcn_readfirstlane(tile_of(max(0, a.causal ? min(p.s.len, before + i0 + 1) : p.s.len) / BN));
    x.low = a.window > 0 && before + i1 - a.window >= 0 ? __builtin_amdgcn_readfirstlane(tile_of((before + i1 - a.window) / BN + 1)) : 0;
    return x;
  };
  const Clear mine = clear_of(r0 + 32 * wave, r0 + 32 * wave + 31), every = clear_of(r0, r_last);
  const int t_up = mine.up, t_low = mine.low;

  s16x8 qf[KS];
  {
    const char* qrow = a.q + (p.s.start + token) * a.q_ts + q_head * a.q_hs + h * 16;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const s16x8*)(qrow + ks * 32);
  }
  // the 1 KB piece of a tile this wave loads: all waves a piece of K and of V each (d = 128), or waves 0-3 the K tile and waves 4-7 the V
  // tile (d = 64)
  const int piece = PIECES == WAVES ? wave : wave & (PIECES - 1);
  const int piece_row = piece * (1024 / ROWB);
  int goff_k, goff_v;
  {
    const int r = lane / CPR, c = lane % CPR;
    goff_k = r * a.c.token_stride + ((c ^ k_swizzle<D>(piece_row + r)) << 4);
    goff_v = r * a.c.token_stride + ((c ^ v_swizzle<D>(piece_row + r)) << 4);
  }
  // a K fragment's offset: that of the first one with the number of its slice in bits that are free (one register, not eight)
  const int koff0 = n * ROWB + ((h ^ k_swizzle<D>(n)) << 4);
  auto koff = [&](int ks) {
    int x = koff0;
    if (ks > 0) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(x) : "n"(32 * ks), "v"(koff0));
    return x;
  };
  int voff[DB];
  {
    const int s = lane & 15, g1 = (lane >> 4) & 1;
    const int row8 = 4 * h + (s >> 2);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int c = 2 * (2 * db + g1) + ((s & 3) >> 1);
      voff[db] = row8 * ROWB + ((c ^ v_swizzle<D>(row8)) << 4) + ((s & 1) << 3);
    }
  }

  // ---- pages: of the 64 tiles that the loads are at and the 64 before them (K runs ahead of V, and the loads of the masks)
  const int* table = a.c.table + (int64_t)p.b * a.c.table_stride;
  int held = -1, page_now = -1, page_prev = -1;               // which 64 tiles; the pages of this wave's piece of them
  uint64_t gone0 = 0, gone1 = 0, gone0_prev = 0, gone1_prev = 0;  // tiles whose first, second 16 keys have no page
  auto hold = [&](int block) {
    HeldPages x;
    const int mine = 64 * block + fresh(lane);
    const bool there = mine < n_tiles;
    x.hold(a.c, table, first_key(mine), there);
    page_prev = page_now;
    gone0_prev = gone0;
    gone1_prev = gone1;
    page_now = max(0, piece_row < 16 ? x.page0 : x.page1);  // page 0 is read in the place of one that is not there, and hidden
    gone0 = __builtin_amdgcn_ballot_w64(there && x.page0 < 0);
    gone1 = __builtin_amdgcn_ballot_w64(there && x.page1 < 0);
    held = block;
  };
  auto hold_for = [&](int t) {  // before the loads of the tiles up to t, at most 63 past those that are held
    if (min(t, n_tiles - 1) >> 6 > held) hold(held + 1);
  };
  auto piece_at = [&](int t) -> int64_t {  // from the start of the pool
    t = min(t, n_tiles - 1);  // loads past the last tile read it again
    const int page = __builtin_amdgcn_readlane(t >> 6 == held ? page_now : page_prev, t & 63);
    return page_row(a.c, page, head, first_key(t) + piece_row);
  };
  auto scalar = [](const char* x) {  // (it is, but the compiler holds it in vector registers where scalar ones run out)
    const uint64_t u = (uint64_t)x;
    return (const char*)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)u) | (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32);
  };
  auto issue_k = [&](int t) {
    if (PIECES < WAVES && wave >= PIECES) return;
    load_lds_16_settled(scalar(a.c.k + piece_at(t)), goff_k, __builtin_amdgcn_readfirstlane(smem_base + (t & (NBUF - 1)) * TILE + piece * 1024));
  };
  auto issue_v = [&](int t) {
    if (PIECES < WAVES && wave < PIECES) return;
    load_lds_16_settled(scalar(a.c.v + piece_at(t)), goff_v, __builtin_amdgcn_readfirstlane(smem_base + (NBUF + (t & (NBUF - 1))) * TILE + piece * 1024));
  };
  auto gone_of = [&](int t) {
    const uint64_t g0 = t >> 6 == held ? gone0 : gone0_prev, g1 = t >> 6 == held ? gone1 : gone1_prev;
    return (int)(g0 >> (t & 63) & 1) | (int)(g1 >> (t & 63) & 1) << 1;
  };
  auto any_gone = [&]() { return ((gone0 | gone1) | (gone0_prev | gone1_prev)) != 0; };
  auto may_be_masked = [&](int t) { return t >= t_up || t < t_low || any_gone(); };
  // which keys this lane's row sees: those below `lim` that are above `low`, or sinks
  struct Sight {
    int lim, low;
  };
  auto sight = [&]() {
    const int t = fresh(token);
    return Sight{a.causal ? min(p.s.len, before + t + 1) : p.s.len, a.window > 0 ? before + t - a.window : -1};
  };
  auto hidden = [&](const Sight& x, int key0, int gone, int e, int hh) {  // is the key of accumulator e of a lane of half hh hidden?
    const int key = key0 + 8 * (e >> 2) + (e & 3) + 4 * hh;
    return bool((key >= x.lim) | ((key <= x.low) & (key >= a.sinks)) | (gone >> (e >> 3) & 1));  // (no branches)
  };

  float m = -INFINITY;  // reference max (raw score units)
  float ms = 0.f;       // m * k2, 0 while m is -inf
  float ls[2] = {0.f, 0.f};
  f32x16 oacc[DB], sacc;  // sacc: scores of the tile in flight, written by an MFMA phase, consumed by the next softmax phase
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  s16x8 pf[2];  // its probabilities in B-operand layout

  auto qk = [&](int kslot) {
    const unsigned char* ks_lds = smem + kslot * TILE;
#pragma unroll
    for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) sacc = E::mma(*(const s16x8*)(ks_lds + koff(ks)), qf[ks], sacc);
  };
  auto mask_tile = [&](int t) {
    if (!may_be_masked(t)) return;
    const int key0 = first_key(t), gone = gone_of(t), half = fresh(lane) >> 5;
    const Sight x = sight();
    if (gone == 0 && key0 >= a.sinks) {  // the keys between `low` and `lim`, as one comparison each
      const unsigned from = key0 + 4 * half - x.low - 1, count = max(0, x.lim - x.low - 1);
#pragma unroll
      for (int e = 0; e < 16; ++e) sacc[e] = from + (8 * (e >> 2) + (e & 3)) < count ? sacc[e] : -INFINITY;
      return;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      sacc[e] = hidden(x, key0, gone, e, half) ? -INFINITY : sacc[e];
  };
  // The reference moves when some row's tile maximum is far above it (or it is unset): until then exponentials may exceed 1, by 2^kLazyLog2.
  auto move_reference = [&]() {
    float m0 = m, m1 = m;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      m0 = fmaxf(fmaxf(m0, sacc[e]), sacc[e + 1]);
      m1 = fmaxf(fmaxf(m1, sacc[e + 2]), sacc[e + 3]);
    }
    const float cand = cross_half_max(fmaxf(m0, m1));
    if (__builtin_amdgcn_ballot_w64((cand - m) * a.scale_log2 > kLazyLog2) != 0) {
      const float cs = (cand == -INFINITY) ? 0.f : cand * a.scale_log2;
      const float alpha = __builtin_amdgcn_exp2f(m * a.scale_log2 - cs);
#pragma unroll
      for (int i = 0; i < 2; ++i) ls[i] *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      m = cand;
      ms = cs;
    }
  };
  // P = exp2(S k2 - m k2); the sums from the unrounded values, the operands of the next product rounded to the storage type: no more than
  // the output's own rounding
  auto softmax_phase = [&]() {
    move_reference();
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
      typename E::vec8 pv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[8 * t2 + e], a.scale_log2, -ms));
        ls[e & 1] += x;
        pv[e] = (typename E::type)x;
      }
      pf[t2] = __builtin_bit_cast(s16x8, pv);
    }
  };
  // A hidden key's probability is 0, and 0 times an infinity or a NaN is not: where the V of a tile that some row has masked holds such
  // a value, the products of masked tiles are taken key by key from there on, over the visible ones.  A wave looks at what it loaded
  // itself, when it has arrived and in front of the barrier behind which the others use it: what it leaves is the pair of tiles that this is the
  // barrier of, since another wave may still have tiles in front of them, whose products are the same whether it has looked yet or not.
  volatile int* odd_from = (volatile int*)(smem + 2 * NBUF * TILE);
  auto look_at_v = [&](int t) {
    if ((PIECES < WAVES && wave < PIECES) || t >= n_tiles || !(t >= every.up || t < every.low || any_gone())) return;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    constexpr unsigned kExp = DT == 0 ? 0x7c007c00u : 0x7f807f80u, kOne = DT == 0 ? 0x04000400u : 0x00800080u;
    const u32x4 x = *(const u32x4*)(smem + (NBUF + (t & (NBUF - 1))) * TILE + piece * 1024 + 16 * fresh(lane));
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top |= (x[e] & kExp) + kOne;  // an exponent of ones carries into the sign's place
    if ((top & 0x80008000u) && *odd_from > t) *odd_from = t & ~1;
  };
  auto odd_values = [&](int t) { return may_be_masked(t) && t >= __builtin_amdgcn_readfirstlane(*odd_from); };
  auto pv_by_key = [&](int t, int vslot) {
    const int key0 = first_key(t), gone = gone_of(t);
    const Sight sees = sight();
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
        if (hidden(sees, key0, gone, e, hh)) continue;
        const float w = hh ? of_upper : of_lower;
        const int half = fresh(lane) >> 5;
        const int key = 8 * (e >> 2) + (e & 3) + 4 * hh;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const typename E::vec4 x =
                *(const typename E::vec4*)(smem + (NBUF + vslot) * TILE + key * ROWB + (((4 * db + q4) ^ v_swizzle<D>(key)) << 4) + 8 * half);
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[db][4 * q4 + i] = __builtin_fmaf(w, (float)x[i], oacc[db][4 * q4 + i]);
          }
      }
    }
  };
  auto phase_fence = [&]() { __builtin_amdgcn_sched_barrier(0); };  // keeps the compiler from mixing the phases
  // The MFMA phase of a tile: O += P(t) V(t), then S(t+1) = K(t+1) Q^T, eight fragment reads ahead of the MFMAs that consume them.
  auto mfma_phase = [&](int vslot, int kslot) __attribute__((always_inline)) {
    phase_fence();
    const unsigned char* vs_lds = smem + (NBUF + vslot) * TILE;
    const unsigned char* ks_lds = smem + kslot * TILE;
    s16x8 vfr[2 * DB], kfr[KS];
    s16x4 half_frag{};
    auto read = [&](int i) {  // halves of the V^T fragments in the order of their MFMAs; then the K fragments
      if (i < 4 * DB) {
        const int f = i / 2;
        const unsigned char* src = vs_lds + 16 * (f / DB) * ROWB + 8 * (i & 1) * ROWB + voff[f % DB];
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(src));
        if (i & 1) vfr[f] = __builtin_shufflevector(half_frag, x, 0, 1, 2, 3, 4, 5, 6, 7);
        else half_frag = x;
      } else if (i < 4 * DB + KS) {
        kfr[i - 4 * DB] = *(const s16x8*)(ks_lds + koff(i - 4 * DB));
      }
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) read(i);
    phase_fence();
#pragma unroll
    for (int f = 0; f < 2 * DB; ++f) {
      oacc[f % DB] = E::mma(vfr[f], pf[f / DB], oacc[f % DB]);
      phase_fence();
      read(8 + 2 * f);
      read(9 + 2 * f);
      phase_fence();
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) sacc = E::mma(kfr[ks], qf[ks], sacc);
  };
  auto ring_barrier = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  // The same in front of tile t, whose V and the next one's it lets in: where masked blocks may follow in some wave.
  auto looking_barrier = [&](int t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    look_at_v(t);
    look_at_v(t + 1);
    __syncthreads();
  };

  // The walk, for one half of the workgroup.  At the start of block t the waves of the first half hold P(t), those of the second half the
  // raw scores S(t).  Block t: the even ones start with the barrier of the pair (t, t+1) -- K(t+1), K(t+2), V(t), V(t+1), issued during
  // the previous pair, have landed, and every wave is past block t-1, so the ring slots of K(t-1), K(t), V(t-2), V(t-1) are free
  // for K(t+3), K(t+4), V(t+2), V(t+3), which are issued during this pair -- then
  //     first half :  O += P(t) V(t), S(t+1) = K(t+1) Q^T  |  softmax of S(t+1)
  //     second half:  softmax of S(t)                      |  O += P(t) V(t), S(t+1) = K(t+1) Q^T
  // Groups of four tiles that need no mask have their ring slots at compile time; the others, and the last few, go tile by tile, and so
  // does everything behind a page that is not there.
  auto walk = [&](auto second_c) __attribute__((always_inline)) {
    constexpr bool SECOND = decltype(second_c)::value;
    auto issue_loads = [&](int t, bool even) __attribute__((always_inline)) {
      if (even) {
        issue_k(t + 3);
        issue_k(t + 4);
      } else {
        issue_v(t + 1);
        issue_v(t + 2);
      }
    };
    auto plain_block = [&](auto slot_c, int t) __attribute__((always_inline)) {
      constexpr int SLOT = decltype(slot_c)::value;  // t mod 4
      if ((SLOT & 1) == 0) ring_barrier();
      if (SECOND) issue_loads(t, (SLOT & 1) == 0);
      phase_fence();
      if (!SECOND) mfma_phase(SLOT, (SLOT + 1) & 3);
      else softmax_phase();
      phase_fence();
      if (!SECOND) issue_loads(t, (SLOT & 1) == 0);
      phase_fence();
      if (!SECOND) softmax_phase();
      else mfma_phase(SLOT, (SLOT + 1) & 3);
      phase_fence();
    };
    auto masked_block = [&](int t) __attribute__((always_inline)) {
      hold_for(t + 4);
      if ((t & 1) == 0) looking_barrier(t);
      if (SECOND) {
        issue_loads(t, (t & 1) == 0);
        softmax_phase();
      }
      phase_fence();
      if (odd_values(t)) {
        pv_by_key(t, t & 3);
        qk((t + 1) & 3);
      } else {
        mfma_phase(t & 3, (t + 1) & 3);
      }
      phase_fence();
      mask_tile(t + 1);
      if (!SECOND) {
        issue_loads(t, (t & 1) == 0);
        if (t + 1 < n_tiles) softmax_phase();  // (the scores past the last tile are of nothing)
      }
      phase_fence();
    };
    mask_tile(0);
    if (!SECOND) softmax_phase();
    // block t has the products of tile t and the scores of tile t + 1.  Three loops one after the other, not one with two ways through it:
    // where two meet again the compiler has two sets of accumulators (64 moves a group, and registers in scratch)
    int t = 0;
    // (by the rows of the workgroup: what a wave does not mask itself it may have to look at for another)
    const int masked_first = min((max(every.low, 0) + 3) & ~3, n_tiles);
#pragma unroll 1
    for (; t < masked_first; ++t) masked_block(t);
#pragma unroll 1
    for (; t + 4 < min(n_tiles, every.up); t += 4) {
      hold_for(t + 6);
      if (any_gone()) break;
      plain_block(std::integral_constant<int, 0>{}, t);
      plain_block(std::integral_constant<int, 1>{}, t + 1);
      plain_block(std::integral_constant<int, 2>{}, t + 2);
      plain_block(std::integral_constant<int, 3>{}, t + 3);
    }
#pragma unroll 1
    for (; t < n_tiles; ++t) masked_block(t);
  };
  if (tid == 0) *odd_from = INT32_MAX;
  if (n_tiles > 0) {
    hold(0);
    issue_k(0);
    issue_k(1);
    issue_k(2);
    issue_v(0);
    issue_v(1);
    __builtin_amdgcn_s_waitcnt(0);  // retire the Q loads with a wait the compiler can see (and the tiles)
    ring_barrier();
    qk(0);
    if (wave < WAVES / 2) walk(std::false_type{});
    else walk(std::true_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // re-reads of the last tile
  }

  const float l = cross_half_sum(ls[0] + ls[1]);
  if (p.splits > 1) {  // as the registers lie: a wave's accumulators as 1 KB a store
    const int64_t slot = (int64_t)(p.slot + p.split) * a.kv_heads + head;
    float* to = a.many.o + (slot * WAVES + wave) * (32 * D) + lane * 4;
#pragma unroll
    for (int i = 0; i < DB * 4; ++i)
      *(f32x4*)(to + 256 * i) = f32x4{oacc[i / 4][i % 4 * 4], oacc[i / 4][i % 4 * 4 + 1], oacc[i / 4][i % 4 * 4 + 2], oacc[i / 4][i % 4 * 4 + 3]};
    if (h == 0) a.many.stat[slot * BM + 32 * wave + n] = float2{l == 0.f ? -INFINITY : ms, l};
    return;
  }
  store_rows<DT, DB>(a, p.s, head, r0 + 32 * wave, r_last, oacc, 0, l, ms);
}

// The shares of a row tile added up in an order of their own: a workgroup has 32 columns of the 32 rows of a wave, its waves every so-many-th
// share.  (A chunk of 16 tokens, 128 K cached, 16 heads on one, 256 shares: 97 us with one wave for all shares and the four column blocks in a
// workgroup, 69, 52 and 51 with two, four and eight waves and a workgroup for each; four sequences of 4 K, 64 tokens each, 8 shares:
// 41, 40, 40 and 47.)  One barrier a call, whatever there is to do.  False behind the last.
template <int DT, int D> static __device__ __forceinline__ bool merge_many(const AttendArgs& a, int block, float (*sums)[18][64]) {
  constexpr int BLOCKS = kManyRows / 32, DB = D / 32;
  const int lane = threadIdx.x & 63, n = lane & 31, sharer = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Place p;
  const int unit = quotient(block, a.by_kv_heads), head = block - unit * a.kv_heads, rows_of = unit / DB % BLOCKS, db = unit % DB;
  if (!find_place<true>(a, unit / (DB * BLOCKS), p)) return false;
  const int r0 = p.tile * kManyRows, r_last = min(r0 + kManyRows, p.s.n * a.group) - 1;
  if (r0 + 32 * rows_of > r_last) {  // (rows of no token: the same for all waves)
    __syncthreads();
    return true;
  }
  const int64_t slot = (int64_t)p.slot * a.kv_heads + head;  // of share 0; those of the others are kv_heads apart
  float top = -INFINITY, l = 0.f;
  f32x16 acc[1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][e] = 0.f;
  auto add = [&](const float2& st, auto of) {
    const float t = fmaxf(top, st.x), keep = t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - t), w = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - t);
    l = __builtin_fmaf(st.y, w, l * keep);
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][e] = __builtin_fmaf(of(e), w, acc[0][e] * keep);
    top = t;
  };
#pragma unroll 4
  for (int s = sharer; s < p.splits; s += kMergeSharers) {
    const int64_t at = slot + (int64_t)s * a.kv_heads;
    const float2 st = a.many.stat[at * kManyRows + 32 * rows_of + n];
    const float* from = a.many.o + (at * BLOCKS + rows_of) * (32 * D) + db * 1024 + lane * 4;
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *(const f32x4*)(from + 256 * i);
    add(st, [&](int e) { return x[e / 4][e % 4]; });
  }
  if (sharer > 0) {
    float (*mine)[64] = sums[sharer - 1];
#pragma unroll
    for (int e = 0; e < 16; ++e) mine[e][lane] = acc[0][e];
    mine[16][lane] = top;
    mine[17][lane] = l;
  }
  __syncthreads();
  if (sharer > 0) return true;
#pragma unroll
  for (int i = 0; i < kMergeSharers - 1; ++i) {
    const float (*x)[64] = sums[i];
    add(float2{x[16][lane], x[17][lane]}, [&](int e) { return x[e][lane]; });
  }
  store_rows<DT, 1>(a, p.s, head, r0 + 32 * rows_of, r_last, acc, db, l, top);
  return true;
}

}  // namespace paged
}  // namespace ringattn
