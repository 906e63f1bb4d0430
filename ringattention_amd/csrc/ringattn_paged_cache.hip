// gfx950 (CDNA4) kernels around the paged cache itself: new rows into it, the attention weight that its tokens have drawn, and the
// eviction that keeps those that drew most.
//
//   paged_append_kernel  : K and V rows of the new tokens to their places.  A copy: 16 bytes a thread.
//   paged_weights_kernel : score[key] += sum over queries of exp(scale q k - LSE).  The sum runs over queries where attention's runs
//       over keys, so a workgroup owns keys: K fragments stay in registers, the query rows pass by, S^T = K Q^T on MFMAs, and a
//       lane adds up the weights of its 16 keys over every 32nd query; lanes meet at the end.  One workgroup adds to a sequence's score, once (an
//       atomic addition, for pages that sequences share): the same bits in every run where they share none.
//   paged_select_kernel  : the places of a sequence's KV head that stay.  The budget-th largest score is found by its bits, from the
//       highest on, in counts of how many scores share the bits so far.
//   paged_present_kernel : takes those whose page is not there out of them, where they are not to stay.
//   paged_move_kernel    : K, V and scores of the kept tokens to the pages of the table that is to hold them.
#include "ringattn_paged.h"

namespace ringattn {
namespace paged {

// ---- append -----------------------------------------------------------------------
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a, int row16, int64_t items) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;  // (token, head, 16 bytes of a row)
  if (item >= items) return;
  const int c16 = (int)(item % row16);
  const int64_t th = item / row16;
  const int head = (int)(th % a.kv_heads), t = (int)(th / a.kv_heads);
  // the sequence that token t is of: the last one that begins at or before it; its lengths and starts are held to the same as everywhere
  int lo = 0, hi = a.c.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.c.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const Seq s = seq_of(a.c, lo);
  const int i = t - s.start, key = s.len - s.n + i;
  if (i < 0 || i >= s.n || key < 0) return;  // in front of the first, behind the last; more new tokens than there are tokens
  const int page = a.c.table[lo * a.c.table_stride + (key >> a.c.page_shift)];
  if ((unsigned)page >= (unsigned)a.c.pages) return;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int64_t from = t * a.ts + head * a.hs + c16 * 16, to = page_row(a.c, page, head, key) + c16 * 16;
  const u32x4 x = *(const u32x4*)(a.k + from), y = *(const u32x4*)(a.v + from);
  *(u32x4*)(a.c.k + to) = x;
  *(u32x4*)(a.c.v + to) = y;
  if (a.scores && c16 == 0) a.scores[(((int64_t)page * a.kv_heads + head) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))] = 0.f;
}

hipError_t launch_paged_append(const AppendArgs& a, int dim, hipStream_t stream) {
  const int64_t items = (int64_t)a.c.tokens * a.kv_heads * (dim / 8);
  if (items <= 0 || a.c.batch <= 0) return hipSuccess;
  const int64_t grid = (items + 255) / 256;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  paged_append_kernel<<<(unsigned)grid, 256, 0, stream>>>(a, dim / 8, items);
  return hipGetLastError();
}

// ---- attention weight of the cached tokens ------------------------------------------
// Where a sequence's KV head has few rows (a.few_most) the waves share out the keys.
// Many: the waves share out the rows, for 128 keys, so that a tile of Q is fetched once for them.
constexpr int kWeightWaves = 8, kWeightPairs = kWeightWaves / 2, kWeightParts = 16, kWeightLaps = 2;

// w[e] of lane (n, h): 16 sums over the 32 lanes of a half at once, each halving of the lanes halving the sums that a lane
// goes on with; lane n ends up with sum n >> 1.  38 instructions for the five steps of 16 separate sums.
static __device__ __forceinline__ float sum_lanes(float (&w)[16]) {
  const int lane = threadIdx.x & 63;
  auto moved = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  using ror8 = std::integral_constant<int, 0x128>;         // within 16 lanes: lane ^ 8
  using half_mirror = std::integral_constant<int, 0x141>;  // within 8: lane ^ 7
  using quad_xor2 = std::integral_constant<int, 0x4e>;
  using quad_xor1 = std::integral_constant<int, 0xb1>;
#pragma unroll
  for (int e = 0; e < 8; ++e) {  // odd rows of 16 lanes go on with w[e + 8]
    // (inline asm: of the builtin's two results the compiler adds one to itself here)
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(w[e]), "+v"(w[e + 8]));
    w[e] += w[e + 8];
  }
  const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = (b3 ? w[e + 4] : w[e]) + moved(b3 ? w[e] : w[e + 4], ror8{});
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = (b2 ? w[e + 2] : w[e]) + moved(b2 ? w[e] : w[e + 2], half_mirror{});
  const float x = (b1 ? w[1] : w[0]) + moved(b1 ? w[0] : w[1], quad_xor2{});
  return x + moved(x, quad_xor1{});
}


// What both kernels know of their sequence and KV head.
template <int DT, int D, int SC> struct WeightRows {
  const WeightsArgs& a;
  const Seq s;
  const int head, rows, before;
  const int* const table;
  const int lane, n, h;
  __device__ __forceinline__ WeightRows(const WeightsArgs& args, const Seq& seq, int b, int head_)
      : a(args), s(seq), head(head_), rows(seq.n * args.group), before(seq.len - seq.n), table(args.c.table + b * args.c.table_stride),
        lane(threadIdx.x & 63), n(lane & 31), h(lane >> 5) {}

  __device__ __forceinline__ void row_of(int r, int& token, int& q_head) const {
    r = min(r, rows - 1);
    token = quotient(r, a.by_group);
    q_head = head * a.group + r - token * a.group;
  }
  __device__ __forceinline__ const char* q_row(int r) const {
    int token, q_head;
    row_of(r, token, q_head);
    return a.q + (s.start + token) * a.q_ts + q_head * a.q_hs;
  }
  __device__ __forceinline__ const float* lse_place(int r) const {
    int token, q_head;
    row_of(r, token, q_head);
    return a.lse + (int64_t)q_head * a.c.tokens + s.start + token;
  }
  // log2(e) LSE of a row; +inf, against which every weight is 0, for a row that is not there or saw nothing
  __device__ __forceinline__ float lse_of(int r) const {
    const float x = *lse_place(r) * 1.4426950408889634f - score_base<SC>(a.x);
    return r >= rows || x == -INFINITY ? INFINITY : x;
  }
  // the new tokens [i0, i1) that see any of the keys [key0, key0 + keys)
  __device__ __forceinline__ void tokens_of(int key0, int keys, int& i0, int& i1) const {
    i0 = a.causal && key0 >= s.prefix ? max(0, key0 - before) : 0;
    i1 = s.n;
    if (a.window > 0 && key0 >= (SC ? max(a.sinks, s.prefix) : a.sinks)) i1 = max(i0, (int)min((int64_t)s.n, (int64_t)key0 + keys - 1 + a.window - before));
  }
  // scores that weigh nothing: of row r, of the 16 keys that a lane has from key0 on.  z: its log2(e) LSE.  One that is no number makes no
  // number of -inf either, so that there the scores of the keys that the row sees are none, and z is 0.
  __device__ __forceinline__ void hide(f32x16& sacc, int key0, int r, float& z) const {
    const float none = z == z ? 0.f : z;
    z = z == z ? z : 0.f;
    const int token = quotient(min(r, rows - 1), a.by_group);
    int lim = r >= rows ? 0 : a.causal ? min(s.len, before + token + 1) : s.len;
    int low = a.window > 0 ? before + token - a.window : -1;
    if constexpr (SC != 0) {
      lim = r >= rows ? 0 : max(lim, s.prefix);
      if (a.x.first) low = max(low, clamped(a.x.first[s.start + token], 0, s.len) - 1);
    }
    if ((SC & kSloped) && s.prefix > 0 && key0 + 31 > before) {
      const int q_head = head * a.group + min(r, rows - 1) - token * a.group;
      turn_slopes(sacc, a.x.slopes[q_head] * 1.4426950408889634f, key0 + 4 * h - before - token, 1.f / unit());
    }
    int first = key0 + 4 * h, sinks = SC ? max(a.sinks, s.prefix) : a.sinks;
    asm volatile("" : "+v"(first), "+v"(sinks));  // (nothing of these comparisons is kept from tile to tile: it took 100 registers)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = first + 8 * (e >> 2) + (e & 3);
      sacc[e] = bool((k >= lim) | ((k <= low) & (k >= sinks))) ? -INFINITY : sacc[e] + none;  // (no branches)
    }
  }
  // What becomes of scores, as in attention, but that a slope goes into what the exponentials take of each (exponent): `at` is slope times the distance of
  // key0 + 4 h, less log2(e) LSE.  A cap first, then masks.
  struct Slope {
    float slope, at;
  };
  __device__ __forceinline__ float unit() const { return shape_unit<SC>(a.x, a.scale_log2); }
  __device__ __forceinline__ void cap(f32x16& sacc) const {
    if constexpr ((SC & kCapped) != 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sacc[e] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(sacc[e] * a.x.cap_in));
    }
  }
  __device__ __forceinline__ float slope_of_row(int r) const {
    int token, q_head;
    row_of(r, token, q_head);
    return a.x.slopes[q_head] * 1.4426950408889634f;
  }
  __device__ __forceinline__ Slope slope_of(int key0, int r, float slope, float z) const {
    if constexpr ((SC & kSloped) == 0) return Slope{0.f, -z};
    return Slope{slope, __builtin_fmaf(slope, (float)(key0 + 4 * h - before - quotient(min(r, rows - 1), a.by_group)), -z)};
  }
  __device__ __forceinline__ float exponent(float s, int e, const Slope& g) const {
    return __builtin_fmaf(s, unit(), (SC & kSloped) ? __builtin_fmaf(g.slope, (float)(8 * (e >> 2) + (e & 3)), g.at) : g.at);
  }
  __device__ __forceinline__ void weigh(float (&w)[16], const f32x16& sacc, const Slope& g) const {
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] += __builtin_amdgcn_exp2f(exponent(sacc[e], e, g));
  }
  // Every key of a sequence has one owner, which adds to its score once: no order to go by.  Atomic, since pages may be several sequences'.
  __device__ __forceinline__ void add_score(int page, int key, float x) const {
    if (page >= 0 && key < s.len)
      unsafeAtomicAdd(a.scores + (((int64_t)page * a.kv_heads + head) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1)), x);
  }
};

// Few rows: a wave has 32 keys at a time, all rows.  Bound by the read of K: tiles come HBM -> LDS one ahead, and every compute unit has eight
// waves of them.
constexpr int kFewWaves = 4;
template <int DT, int D, int SC>
__global__ __launch_bounds__(64 * kFewWaves, 2) void paged_weights_few_kernel(const WeightsArgs a) {
  using E = Elem<DT>;
  constexpr int KS = D / 16, ROWB = D * 2, TILE = 32 * ROWB, HALF = D / 32;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kFewWaves * 2 * TILE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x, b = blockIdx.z;
  const Seq s = uniform(seq_of(a.c, b, SC ? a.x.prefix : nullptr));
  const WeightRows<DT, D, SC> x(a, s, b, head);
  if (x.rows == 0 || s.len == 0 || x.rows > a.few_most) return;
  const int n = x.n, h = x.h;
  const Keys keys = keys_of(s, 0, s.n - 1, a.causal, a.window, a.sinks, SC ? firsts_of(a.x, s, 0, s.n - 1).least : 0);  // that any row sees
  const int tiles = keys.count, step = gridDim.y * kFewWaves;
  auto first_key = [&](int u) { return (u < keys.sink_tiles ? u : u + keys.skip) * kKeyTile; };
  int u = blockIdx.y * kFewWaves + wave;
  if (u >= tiles) return;
  // the first 32 rows stay in registers
  s16x8 qf[KS];
  {
    const char* q = x.q_row(n) + h * 16;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const s16x8*)(q + ks * 32);
  }
  const float lse_first = x.lse_of(n), slope_first = (SC & kSloped) ? x.slope_of_row(n) : 0.f;
  unsigned char* my = smem + wave * 2 * TILE;
  const unsigned my_lds = lds_offset(smem) + wave * 2 * TILE;
  int koff[KS], goff[HALF];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = n * ROWB + (((2 * ks + h) ^ k_swizzle<D>(n)) << 4);
  half_tile_offsets<D>(goff, a.c.token_stride, [](int r) { return k_swizzle<D>(r); });
  HeldPages held;
  int held_from = u;
  auto hold = [&](int first) {
    held_from = first;
    held.hold(a.c, x.table, first_key(first + step * x.lane), first + step * x.lane < tiles);
  };
  hold(u);
  int at = 0, p0, p1, next0 = 0, next1 = 0;  // place of tile u among the held ones; its pages
  auto issue = [&](int key, int slot, int page0, int page1) {
    load_half_tile<true>(a.c.k + page_row(a.c, max(page0, 0), head, key), my_lds + slot * TILE, goff);
    load_half_tile<true>(a.c.k + page_row(a.c, max(page1, 0), head, key + 16), my_lds + slot * TILE + TILE / 2, goff);
  };
  p0 = __builtin_amdgcn_readlane(held.page0, 0);
  p1 = __builtin_amdgcn_readlane(held.page1, 0);
  __builtin_amdgcn_s_waitcnt(0);
  issue(first_key(u), 0, p0, p1);
  for (int slot = 0; u < tiles; u += step, slot ^= 1, p0 = next0, p1 = next1) {
    const int key0 = first_key(u);
    if (u + step < tiles) {
      if (++at == 64) {
        hold(u + step);
        at = 0;
      }
      next0 = __builtin_amdgcn_readlane(held.page0, at);
      next1 = __builtin_amdgcn_readlane(held.page1, at);
      issue(first_key(u + step), slot ^ 1, next0, next1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * HALF) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    s16x8 kfr[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kfr[ks] = *(const s16x8*)(my + slot * TILE + koff[ks]);
    float w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = 0.f;
    {
      f32x16 sacc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sacc = E::mma(kfr[ks], qf[ks], sacc);
      float z = lse_first;
      x.cap(sacc);
      x.hide(sacc, key0, n, z);
      x.weigh(w, sacc, x.slope_of(key0, n, slope_first, z));
    }
#pragma unroll 1
    for (int r0 = 32; r0 < x.rows; r0 += 32) {
      const char* q = x.q_row(r0 + n) + h * 16;
      float z = x.lse_of(r0 + n);
      f32x16 sacc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sacc = E::mma(kfr[ks], *(const s16x8*)(q + ks * 32), sacc);
      x.cap(sacc);
      x.hide(sacc, key0, r0 + n, z);
      x.weigh(w, sacc, x.slope_of(key0, r0 + n, (SC & kSloped) ? x.slope_of_row(r0 + n) : 0.f, z));
    }
    const float sum = sum_lanes(w);
    const int e = n >> 1;
    if ((n & 1) == 0) x.add_score(e < 8 ? p0 : p1, key0 + 8 * (e >> 2) + (e & 3) + 4 * h, sum);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// Many rows: a workgroup has 128 keys and some of the rows that see them, kWeightPairs tiles of 32 rows at a time; two waves share a
// tile, 64 keys each.  Q and LSE come to LDS two steps ahead, and while a wave's products of one tile are on the matrix cores it has the
// exponentials of the tile before: 16 MFMAs of 32 cycles to 32 x (fma 4, exp 8, add 4) cycles of vector arithmetic, which the two share a SIMD's
// issue for.  A prompt of 8 K tokens, 16/4 heads of 128, causal: 160 us, 860 TFLOP/s (250 with every tile's places worked out, 202 with
// a Q tile for each wave and nothing on the way while it has the exponentials, 180 with no equal shares of the triangle).  Bound by power as much as
// by the order of things: with queries and keys of 0 the same launch takes 140 us.  Workgroups of four waves, two to a compute unit, take
// 162: of two waves of a SIMD that wait for nothing together the older one gets most of its issue, and when it is done the younger is alone.
template <int DT, int D, int SC>
__global__ __launch_bounds__(64 * kWeightWaves, 2) void paged_weights_kernel(const WeightsArgs a) {
  using E = Elem<DT>;
  constexpr int KS = D / 16, ROWB = D * 2, TILE = 32 * ROWB, CPR = D / 8, PIECES = TILE / 2048;  // (pieces of 1 KB that a wave brings of its tile)
  constexpr int STEP = 32 * kWeightPairs;
  constexpr int LSES = kWeightPairs * TILE, SLOT = LSES + kWeightWaves * 256;  // of a step: tiles; LSEs, a lane's own
  __shared__ __attribute__((aligned(1024))) unsigned char smem[3 * SLOT];
  __shared__ float part[kWeightPairs][kManyKeys];
  __shared__ int last;
  __shared__ Firsts ends[SC ? kWeightWaves : 1];
  __shared__ int see_all[SC ? kWeightWaves : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, pair = wave >> 1, half = wave & 1;
  const int head = blockIdx.x, block = blockIdx.y, in_all = gridDim.y;
  // the blockIdx.z-th sequence of many rows: there are fewer of them than sequences
  int b = -1;
  Seq s{};
  for (int b0 = 0, before = 0; b0 < a.c.batch && b < 0; b0 += 64) {
    Seq mine{};
    if (b0 + lane < a.c.batch) mine = seq_of(a.c, b0 + lane, SC ? a.x.prefix : nullptr);
    const uint64_t many = __builtin_amdgcn_ballot_w64(mine.n * a.group > a.few_most);
    const int wanted = (int)blockIdx.z - before, count = __builtin_popcountll(many);
    if (wanted < count) {
      const bool it = (many >> lane & 1) && __builtin_popcountll(many & (((uint64_t)1 << lane) - 1)) == wanted;
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(it));
      s = Seq{__builtin_amdgcn_readlane(mine.len, l), __builtin_amdgcn_readlane(mine.start, l), __builtin_amdgcn_readlane(mine.n, l),
              SC ? __builtin_amdgcn_readlane(mine.prefix, l) : 0};
      b = b0 + l;
    }
    before += count;
  }
  if (b < 0) return;
  const WeightRows<DT, D, SC> x(a, s, b, head);
  const int n = x.n, h = x.h, before = x.before;
  auto page_of = [&](int key) {  // -1: not there, or behind the end
    const int page = key < s.len ? x.table[key >> a.c.page_shift] : -1;
    return (unsigned)page < (unsigned)a.c.pages ? page : -1;
  };
  const unsigned q_lds = lds_offset(smem) + pair * TILE + half * (PIECES * 1024), lse_lds = lds_offset(smem) + LSES + wave * 256;
  const int qoff = pair * TILE + n * ROWB + ((h ^ k_swizzle<D>(n)) << 4);
  // A tile of Q, 1 KB a piece, half of them by each of the two waves.  Where 32 rows are whole tokens (a.q_even) a piece's rows lie at
  // fixed offsets from the tile's first, and so do the rows of their LSEs; elsewhere, and where the last rows are not there, every row's
  // place is worked out.  (Worked out for every tile it cost as much as the exponentials: a prompt of 8 K tokens, 16/4 heads 250 us.)
  // (Rows of a lane are then of one head, whose slope stays in a register.)
  const float even_slope = (SC & kSloped) && a.q_even ? x.slope_of_row(n) : 0.f;
  int at_piece[PIECES], lse_at = 0;
#pragma unroll
  for (int j = 0; j < PIECES; ++j) at_piece[j] = 0;
  if (a.q_even) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int r = 1024 / ROWB * (half * PIECES + j) + lane / CPR, token = quotient(r, a.by_group);
      at_piece[j] = (int)(token * a.q_ts + (r - token * a.group) * a.q_hs) + (((lane % CPR) ^ k_swizzle<D>(r)) << 4);
    }
    const int token = quotient(n, a.by_group);
    lse_at = ((n - token * a.group) * a.c.tokens + token) * 4;
  }
  const int64_t q_step = (int64_t)quotient(STEP, a.by_group) * a.q_ts;
  const int lse_step = quotient(STEP, a.by_group);
  // Blocks of keys; where there are workgroups enough, each block's rows are cut into as many parts, whose sums the last one to be done adds up,
  // in their order.  Under the mask the first blocks are seen by the most rows, and laps over the blocks go to and fro.
  int blocks = (s.len + kManyKeys - 1) / kManyKeys;
  // Of a scored call only those that some row sees, if all documents and windows are looked at together: the first ones, and those behind `passed` more.
  // (Eight sequences of 5 to 58 K tokens, some 100 new ones each, 16/4 heads x 64 and a window of 257: 115 us through all blocks, 30 so.)
  int front = blocks, passed = 0;
  if constexpr (SC != 0) {
    int least = 0;
    if (a.x.first) {
      least = s.len;
      for (int i = (int)threadIdx.x; i < s.n; i += 64 * kWeightWaves) least = min(least, max(a.x.first[s.start + i], 0));
      const Firsts here = firsts_of_lanes(least, least);
      if (lane == 0) ends[wave] = here;
      __syncthreads();
      for (int i = 0; i < kWeightWaves; ++i) least = min(least, ends[i].least);
      least = __builtin_amdgcn_readfirstlane(least);
    }
    constexpr int EACH = kManyKeys / kKeyTile;
    const Keys keys = keys_of(s, 0, s.n - 1, a.causal, a.window, a.sinks, least);
    front = (keys.sink_tiles + EACH - 1) / EACH;
    passed = max(0, (keys.sink_tiles + keys.skip) / EACH - front);
    blocks = max(0, (keys.count + keys.skip + EACH - 1) / EACH - passed);
  }
  const bool room = (int)(gridDim.x * gridDim.z) * in_all <= kWeightUnits / kWeightLaps;  // for all parts' sums
  const int parts = room ? clamped(min(kWeightLaps * in_all / max(blocks, 1), x.rows / (4 * STEP)), 1, kWeightParts) : 1;
  for (int lap = 0; lap * in_all < blocks * parts; ++lap) {
    const int unit = lap * in_all + (lap & 1 ? in_all - 1 - block : block);
    if (unit >= blocks * parts) continue;
    const int at = unit / parts, my_part = unit - at * parts;
    const int key0 = (SC != 0 && at >= front ? at + passed : at) * kManyKeys, my_key0 = key0 + 64 * half;
    int i0, i1;
    x.tokens_of(key0, kManyKeys, i0, i1);
    bool hides = false;  // whether some of these tokens may not see some of these keys for their documents' sake
    if constexpr (SC != 0) {
      // Of documents, the tokens between the first and the last that see any of these keys: one look at where all of theirs begin.  (16 K tokens in
      // documents of 1365, 16/4 heads: 1136 us without, 220 with it.  Blocks in which no document begins are compared as those of plain calls are: all
      // 16 K tokens one document 666 us, 1136 with a comparison for every key; plain 620.)
      if (a.x.first && key0 >= max(a.sinks, s.prefix)) {
        int least = i1, most = i0 - 1, count = 0;
        for (int i = i0 + (int)threadIdx.x; i < i1; i += 64 * kWeightWaves) {
          const int f = a.x.first[s.start + i];
          if (f >= key0 + kManyKeys) continue;
          least = min(least, i);
          most = max(most, i);
          count += f <= key0;
        }
        const Firsts here = firsts_of_lanes(least, most);
        count = wave_sum(count);
        __syncthreads();
        if (lane == 0) {
          ends[wave] = here;
          see_all[wave] = count;
        }
        __syncthreads();
        least = ends[0].least;
        most = ends[0].most;
        count = see_all[0];
        for (int i = 1; i < kWeightWaves; ++i) {
          least = min(least, ends[i].least);
          most = max(most, ends[i].most);
          count += see_all[i];
        }
        i0 = __builtin_amdgcn_readfirstlane(least);
        i1 = max(i0, __builtin_amdgcn_readfirstlane(most) + 1);
        hides = __builtin_amdgcn_readfirstlane(count) < i1 - i0;
      } else {
        hides = a.x.first != nullptr;
      }
    }
    if (SC != 0 && i1 <= i0) continue;  // (seen by none: the same for all parts)
    const int r_begin = i0 * a.group, steps = max(0, (i1 - i0) * a.group + STEP - 1) / STEP;
    int t = my_part * steps / parts;
    const int t_end = (my_part + 1) * steps / parts;
    // steps whose rows are all there and lie evenly, and the first of them
    const int even_end = a.q_even ? (x.rows - r_begin) / STEP : 0;
    const int first_token = s.start + quotient(r_begin + t * STEP + 32 * pair, a.by_group);
    const char* q_next = a.q + first_token * a.q_ts + (int64_t)head * a.group * a.q_hs;
    const float* lse_next = a.lse + (int64_t)head * a.group * a.c.tokens + first_token;
    auto fetch = [&](int step, int to) {  // PIECES + 1 loads; steps come in their order
      if (step < even_end) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) load_lds_16_settled(q_next, at_piece[j], q_lds + to + 1024 * j);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(lse_lds + to), "v"(lse_at), "s"(lse_next) : "m0");
        q_next += q_step;
        lse_next += lse_step;
        return;
      }
      const int r0 = r_begin + step * STEP + 32 * pair;
#pragma unroll 1
      for (int j = 0; j < PIECES; ++j) {
        const int r = 1024 / ROWB * (half * PIECES + j) + lane / CPR;
        const char* src = x.q_row(r0 + r) + (((lane % CPR) ^ k_swizzle<D>(r)) << 4);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(q_lds + to + 1024 * j), "v"(src) : "m0");
      }
      const float* lse = x.lse_place(r0 + n);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, off" ::"s"(lse_lds + to), "v"(lse) : "m0");
    };
    // the steps all of whose rows see all of the keys
    int seen_from = 0, seen_to = (SC && a.x.first ? (i1 - i0) * a.group : x.rows - r_begin) / STEP;  // (rows of later documents see none)
    if (a.causal) seen_from = (max(0, key0 + kManyKeys - 1 - before - i0) * a.group + STEP - 1) / STEP;
    if (key0 + kManyKeys > s.len || hides) seen_to = 0;
    if (a.window > 0 && key0 + kManyKeys > a.sinks) seen_to = min(seen_to, (int)max((int64_t)0, min((int64_t)s.n, (int64_t)key0 + a.window - before - i0)) * a.group / STEP);
    const unsigned seen = max(0, seen_to - seen_from);
    s16x8 kfr[2][KS];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = my_key0 + 32 * c + n;
      const char* src = a.c.k + page_row(a.c, max(page_of(key), 0), head, key) + h * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kfr[c][ks] = *(const s16x8*)(src + ks * 32);
    }
    float w[2][16];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) w[c][e] = 0.f;
    int here = 0, next = SLOT, free = 2 * SLOT;
    // Tile t's products.  Every wave's own loads of it have come before the barrier, so behind it all have; and behind it all have read the
    // tile before, whose slot takes the one two steps ahead.
    s16x8 qfr[KS];
    auto receive = [&](float& z) {
      if (t + 1 < t_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PIECES + 1) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const int from = here + qoff;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {  // (the number of the slice in bits that are free: one register, not eight)
        int o = from;
        if (ks > 0) asm volatile("v_xor_b32 %0, %1, %2" : "=v"(o) : "n"(32 * ks), "v"(from));
        qfr[ks] = *(const s16x8*)(smem + o);
      }
      const float raw = *(const float*)(smem + here + LSES + threadIdx.x * 4) * 1.4426950408889634f - score_base<SC>(a.x);
      z = raw == -INFINITY ? INFINITY : raw;
      if (t + 2 < t_end) fetch(t + 2, free);
      const int last = free;
      free = here;
      here = next;
      next = last;
    };
    auto multiply = [&](f32x16 (&sacc)[2]) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) sacc[c][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int c = 0; c < 2; ++c) sacc[c] = E::mma(kfr[c][ks], qfr[ks], sacc[c]);
    };
    auto hide = [&](f32x16 (&sacc)[2], int step, float& z) {
#pragma unroll
      for (int c = 0; c < 2; ++c) x.cap(sacc[c]);
      if ((unsigned)(step - seen_from) >= seen) {
        const float from = z;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          z = from;
          x.hide(sacc[c], my_key0 + 32 * c, r_begin + step * STEP + 32 * pair + n, z);
        }
      }
    };
    using Slope = typename WeightRows<DT, D, SC>::Slope;
    // of a step that has been through hide()
    auto weigh = [&](const f32x16 (&sacc)[2], const Slope (&g)[2]) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          w[c][e] += __builtin_amdgcn_exp2f(x.exponent(sacc[c][e], e, g[c]));
          asm volatile("" : "+v"(w[c][e]));  // (here, not where the sums are used next)
        }
    };
    auto slopes = [&](Slope (&g)[2], int step, float z) {
      const int r = r_begin + step * STEP + 32 * pair + n;
      float slope = even_slope;
      if ((SC & kSloped) && !a.q_even) slope = x.slope_of_row(r);
#pragma unroll
      for (int c = 0; c < 2; ++c) g[c] = x.slope_of(my_key0 + 32 * c, r, slope, z);
    };
    auto both = [&](f32x16 (&next)[2], float& z_next, f32x16 (&sacc)[2], float z) {
      receive(z_next);
      hide(sacc, t - 1, z);
      Slope g[2];
      slopes(g, t - 1, z);
      __builtin_amdgcn_sched_barrier(0);
      multiply(next);
      weigh(sacc, g);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, ((SC & kSloped) ? 48 : 32) / KS, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 16 / KS, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto last_one = [&](f32x16 (&sacc)[2], int step, float z) {
      hide(sacc, step, z);
      Slope g[2];
      slopes(g, step, z);
      weigh(sacc, g);
    };
    if (t < t_end) {
      fetch(t, here);
      if (t + 1 < t_end) fetch(t + 1, next);
      f32x16 odd[2], even[2];
      float z_odd, z_even;
      receive(z_even);
      multiply(even);
      for (++t; t + 1 < t_end; t += 2) {
        both(odd, z_odd, even, z_even);
        ++t;
        both(even, z_even, odd, z_odd);
        --t;
      }
      if (t < t_end) {
        both(odd, z_odd, even, z_even);
        last_one(odd, t, z_odd);
      } else {
        last_one(even, t - 1, z_even);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float sum = sum_lanes(w[c]);
      const int e = n >> 1;
      if ((n & 1) == 0) part[pair][64 * half + 32 * c + 8 * (e >> 2) + (e & 3) + 4 * h] = sum;
    }
    __syncthreads();
    float sum = 0.f;
    if (threadIdx.x < kManyKeys) {
#pragma unroll
      for (int i = 0; i < kWeightPairs; ++i) sum += part[i][threadIdx.x];
    }
    if (parts > 1) {  // (of no more units than kWeightLaps laps)
      const int first = (blockIdx.z * gridDim.x + head) * kWeightLaps * in_all + at * parts;
      if (threadIdx.x < kManyKeys)
        __hip_atomic_store(a.parts + (int64_t)(first + my_part) * kManyKeys + threadIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (threadIdx.x == 0) {
        last = __hip_atomic_fetch_add(a.arrived + first, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        if (last) __hip_atomic_store(a.arrived + first, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
      }
      __syncthreads();
      if (!last) continue;
      if (threadIdx.x < kManyKeys) {
        sum = 0.f;
        for (int i = 0; i < parts; ++i)
          sum += __hip_atomic_load(a.parts + (int64_t)(first + i) * kManyKeys + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    if (threadIdx.x < kManyKeys) x.add_score(page_of(key0 + threadIdx.x), key0 + threadIdx.x, sum);
    __syncthreads();
  }
}

template <int SC> static hipError_t launch_weights(const WeightsArgs& a, int dtype, int dim, hipStream_t stream) {
  const int64_t keys = (int64_t)a.c.table_pages << a.c.page_shift;
  const int64_t pairs = (int64_t)a.c.batch * a.kv_heads;
  if (pairs <= 0 || keys <= 0) return hipSuccess;
  if (a.c.batch > 65535) return hipErrorInvalidValue;
  // A launch for the sequences of few rows and one for those of many, where there may be any; one sequence has one of the two, whichever its
  // rows turn out to be (ringattn_paged_weights).  As many workgroups as the longest sequence could use, where that does not make them more
  // than enough: they go on to further keys.  (Of many rows, 256 for one sequence, all of which has equal shares; of several, any may have few
  // rows and leave its workgroups idle: 85 sequences of some 1 K tokens, ten of which have 60 to 100 new ones, 16 heads on 2: 181 us with
  // 256, 62 with 1024.)
  const int64_t rows = (int64_t)a.c.tokens * a.group;
  auto grid = [&](int keys_each, int64_t sequences, int64_t enough) {
    const int64_t blocks = (keys + keys_each - 1) / keys_each, each = enough / (sequences * a.kv_heads);
    return dim3((unsigned)a.kv_heads, (unsigned)(blocks < each ? blocks : each > 1 ? each : 1), (unsigned)sequences);
  };
  const int64_t might = rows / ((int64_t)a.few_most + 1), with_many = might < a.c.batch ? might : a.c.batch;
#define RA_LAUNCH_WEIGHTS(DT_, D_)                                                                                                      \
  do {                                                                                                                                 \
    if (a.c.batch > 1 || with_many == 0)                                                                                               \
      paged_weights_few_kernel<DT_, D_, SC><<<grid(kFewWaves * kKeyTile, a.c.batch, 2048), 64 * kFewWaves, 0, stream>>>(a);                 \
    if (with_many > 0)                                                                                                                 \
      paged_weights_kernel<DT_, D_, SC>                                                                                                \
          <<<grid(kManyKeys / kWeightParts, with_many, with_many > 1 ? kWeightUnits / kWeightLaps : 256), 64 * kWeightWaves, 0, stream>>>(a); \
  } while (0)
  if (dtype == 0 && dim == 64) RA_LAUNCH_WEIGHTS(0, 64);
  else if (dtype == 1 && dim == 64) RA_LAUNCH_WEIGHTS(1, 64);
  else if (dtype == 0 && dim == 128) RA_LAUNCH_WEIGHTS(0, 128);
  else if (dtype == 1 && dim == 128) RA_LAUNCH_WEIGHTS(1, 128);
#undef RA_LAUNCH_WEIGHTS
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_paged_weights(const WeightsArgs& a, int sc, int dtype, int dim, hipStream_t stream) {
  switch (sc) {
    case 0: return launch_weights<0>(a, dtype, dim, stream);
    case kScored: return launch_weights<kScored>(a, dtype, dim, stream);
    case kScored | kCapped: return launch_weights<kScored | kCapped>(a, dtype, dim, stream);
    case kScored | kSloped: return launch_weights<kScored | kSloped>(a, dtype, dim, stream);
    case kScored | kCapped | kSloped: return launch_weights<kScored | kCapped | kSloped>(a, dtype, dim, stream);
  }
  return hipErrorInvalidValue;
}

// ---- eviction ----------------------------------------------------------------------
// Larger scores have larger ranks; a NaN ranks with -inf, and so does a token whose page is not there, or below it where such are not to stay.
static __device__ __forceinline__ unsigned rank_of(float x) {
  if (!(x == x)) x = -INFINITY;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);  // (-0 as 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kDigit = 11, kBins = 1 << kDigit, kPasses = 3;
constexpr int kHeld = 8;  // ranks that a thread keeps in registers from pass to pass; those beyond are read again
// Bits of digit `pass` of a rank, from the highest on, and where they begin.
static __device__ __forceinline__ constexpr int digit_bits(int pass) { return pass < 2 ? kDigit : 32 - 2 * kDigit; }
static __device__ __forceinline__ constexpr int digit_shift(int pass) { return pass == 0 ? 32 - kDigit : pass == 1 ? 32 - 2 * kDigit : 0; }

// What is known of the rank of the last token that stays: its digits so far, and how many of those that share them stay.
struct Found {
  unsigned prefix, wanted;
};

// A slice of a sequence's KV head: its tokens whose scores decide, and their ranks.
struct Slice {
  int begin, end;
  unsigned held[kHeld];
};
// Ranks of up to kHeld tokens of a thread, from key0 on.  All pages first, then all scores, with nothing in between that a lane might skip.
static __device__ __forceinline__ void load_ranks(const EvictArgs& a, const int* table, int head, int key0, int end, unsigned (&r)[kHeld]) {
  const int mask = (1 << a.c.page_shift) - 1;
  const unsigned gone = a.present ? 0 : rank_of(-INFINITY);
  auto key_at = [&](int i) { return max(min(key0 + i * kSelectThreads + (int)threadIdx.x, end - 1), 0); };
  int page[kHeld];
  float x[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) page[i] = table[key_at(i) >> a.c.page_shift];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int there = (unsigned)page[i] < (unsigned)a.c.pages ? page[i] : 0;
    x[i] = a.scores[(((int64_t)there * a.kv_heads + head) << a.c.page_shift) + (key_at(i) & mask)];
  }
#pragma unroll
  for (int i = 0; i < kHeld; ++i) r[i] = (unsigned)page[i] < (unsigned)a.c.pages ? rank_of(x[i]) : gone;
}
// fn(first key, ranks) for every kHeld x kSelectThreads tokens of a slice
template <class Fn> static __device__ __forceinline__ void each_ranks(const EvictArgs& a, const int* table, int head, Slice& s, bool first, Fn fn) {
  if (first) load_ranks(a, table, head, s.begin, s.end, s.held);
  fn(s.begin, s.held);
  for (int key0 = s.begin + kHeld * kSelectThreads; key0 < s.end; key0 += kHeld * kSelectThreads) {
    unsigned r[kHeld];
    load_ranks(a, table, head, key0, s.end, r);
    fn(key0, r);
  }
}

// How many of a slice's ranks that begin with `prefix` have each value of the digit behind it.
static __device__ __forceinline__ void count_digits(const EvictArgs& a, const int* table, int head, Slice& s, bool first, int pass, unsigned prefix,
                                                    unsigned* counts) {
  const int lane = threadIdx.x & 63, shift = digit_shift(pass), bits = digit_bits(pass);
  const unsigned known = pass == 0 ? 0 : ~0u << (shift + bits);
  for (int i = threadIdx.x; i < kBins; i += kSelectThreads) counts[i] = 0;
  __syncthreads();
  each_ranks(a, table, head, s, first, [&](int key0, const unsigned (&ranks)[kHeld]) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const unsigned r = ranks[i];
      const bool counted = key0 + i * kSelectThreads + (int)threadIdx.x < s.end && (r & known) == prefix;
      const unsigned digit = r >> shift & ((1u << bits) - 1);
      // scores that drew nothing all have one rank: the lanes that share the first one's digit are one addition
      const uint64_t any = __builtin_amdgcn_ballot_w64(counted);
      if (any == 0) continue;
      const int one = __builtin_ctzll(any);
      const unsigned lead = __builtin_amdgcn_readlane(digit, one);
      const uint64_t same = __builtin_amdgcn_ballot_w64(counted && digit == lead);
      if (lane == one) atomicAdd(&counts[lead], (unsigned)__builtin_popcountll(same));
      else if (counted && digit != lead) atomicAdd(&counts[digit], 1u);
    }
  });
  __syncthreads();
}

// The digit at which the counts, added up from the highest value on, reach f.wanted; a thread has the counts of two values, `c0` of the
// higher one.  `shared`: room for a number of every wave and two more.
static __device__ __forceinline__ void find_digit(unsigned c0, unsigned c1, int pass, Found& f, unsigned* shared) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = kBins - 1 - 2 * (int)threadIdx.x;
  const int both = (int)(c0 + c1), upto = wave_scan(both);
  if (lane == 63) shared[wave] = upto;
  __syncthreads();
  const int above = upto - both + wave_sum(lane < wave ? (int)shared[lane] : 0);  // (of the waves in front)
  const int want = (int)f.wanted;
  unsigned* found = shared + kSelectThreads / 64;
  if (above < want && want <= above + (int)c0) {
    found[0] = hi;
    found[1] = above;
  } else if (above + (int)c0 < want && want <= above + both) {
    found[0] = hi - 1;
    found[1] = above + c0;
  }
  __syncthreads();
  f.prefix |= found[0] << digit_shift(pass);
  f.wanted -= found[1];
  __syncthreads();
}

// Places of the tokens [begin, end) that stay, in order, from kept[placed] on: those outside [from, to), those that rank above
// f.prefix, and of those that rank the same the first ones while fewer than f.wanted came before.
static __device__ __forceinline__ void place_tokens(const EvictArgs& a, const int* table, int head, Slice& s, bool first, int* kept, int placed,
                                                    int equal_before, const Found& f, unsigned* counts) {
  static_assert(kHeld * (kSelectThreads / 64) == 128, "two of them a lane");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wanted = (int)f.wanted;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  each_ranks(a, table, head, s, first, [&](int key0, const unsigned (&r)[kHeld]) {
    // how many of 64 tokens rank above (low 16 bits) and the same (high), 64 after 64, and of all in front of them
    uint64_t mores[kHeld], sames[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const bool there = key0 + i * kSelectThreads + (int)threadIdx.x < s.end && wanted > 0;
      mores[i] = __builtin_amdgcn_ballot_w64(there && r[i] > f.prefix);
      sames[i] = __builtin_amdgcn_ballot_w64(there && r[i] == f.prefix);
      if (lane == 0) counts[i * (kSelectThreads / 64) + wave] = (unsigned)__builtin_popcountll(sames[i]) << 16 | (unsigned)__builtin_popcountll(mores[i]);
    }
    __syncthreads();
    const int x0 = (int)counts[lane], x1 = (int)counts[64 + lane], s0 = wave_scan(x0), s1 = wave_scan(x1);
    __syncthreads();
    const unsigned first64 = __builtin_amdgcn_readlane(s0, 63), all = first64 + __builtin_amdgcn_readlane(s1, 63);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int at64 = i * (kSelectThreads / 64) + wave;
      const unsigned front = at64 < 64 ? __builtin_amdgcn_readlane(s0 - x0, at64) : first64 + __builtin_amdgcn_readlane(s1 - x1, at64 - 64);
      const int eq = equal_before + (int)(front >> 16) + __builtin_popcountll(sames[i] & below);  // those that rank the same in front of this one
      const int ab = (int)(front & 0xffff) + __builtin_popcountll(mores[i] & below);
      const int at = placed + ab + min(eq, wanted) - min(equal_before, wanted);
      const bool stays = (mores[i] >> lane & 1) || ((sames[i] >> lane & 1) && eq < wanted);
      if (stays && at < a.budget) kept[at] = key0 + i * kSelectThreads + (int)threadIdx.x;
    }
    placed += (int)(all & 0xffff) + min(equal_before + (int)(all >> 16), wanted) - min(equal_before, wanted);
    equal_before += all >> 16;
  });
}

// What every workgroup of a selection begins with.  The slices of [from, to) have as many tokens each.
struct Selection {
  int len, from, to;
  int* kept;
  const int* table;
  Slice s;
  unsigned wanted;
};
static __device__ __forceinline__ Selection selection_of(const EvictArgs& a, int head, int b, int slice, int slices) {
  Selection x;
  x.len = __builtin_amdgcn_readfirstlane(clamped(a.c.lens[b], 0, a.c.table_pages << a.c.page_shift));
  x.kept = a.kept + ((int64_t)b * a.kv_heads + head) * a.budget;
  x.table = a.c.table + b * a.c.table_stride;
  x.from = a.first;
  x.to = x.len - a.last;
  const int count = x.to - x.from, each = ((count + slices - 1) / slices + 63) & ~63;
  x.s.begin = min(x.to, x.from + slice * each);
  x.s.end = min(x.to, x.s.begin + each);
  x.wanted = a.budget - a.first - a.last;
  return x;
}
// The first and the last tokens, or all of a sequence that is short enough; the end of the list.  True if there is more to select.
static __device__ __forceinline__ bool place_ends(const EvictArgs& a, const Selection& x) {
  const int tid = threadIdx.x, stay = min(x.len, a.budget);
  for (int j = stay + tid; j < a.budget; j += kSelectThreads) x.kept[j] = -1;
  if (x.len <= a.budget) {
    for (int j = tid; j < x.len; j += kSelectThreads) x.kept[j] = j;
    return false;
  }
  for (int j = tid; j < a.first; j += kSelectThreads) x.kept[j] = j;
  for (int j = tid; j < a.last; j += kSelectThreads) x.kept[a.budget - a.last + j] = x.len - a.last + j;
  return x.wanted > 0;
}

// One workgroup for a sequence's KV head: all passes, the ranks of up to 8 K tokens in registers.
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(const EvictArgs a) {
  __shared__ unsigned counts[kBins];
  __shared__ unsigned shared[kSelectThreads / 64 + 2];
  const int head = blockIdx.x, b = blockIdx.y, hi = kBins - 1 - 2 * (int)threadIdx.x;
  Selection x = selection_of(a, head, b, 0, 1);
  if (!place_ends(a, x)) return;
  Found f{0, x.wanted};
  for (int pass = 0; pass < kPasses; ++pass) {
    count_digits(a, x.table, head, x.s, pass == 0, pass, f.prefix, counts);
    find_digit(counts[hi], counts[hi - 1], pass, f, shared);
  }
  place_tokens(a, x.table, head, x.s, false, x.kept, a.first, 0, f, counts);
}

// The same by several workgroups, where there are few sequences and heads and they are long: a launch for each pass, in which
// every workgroup adds up the counts that the launch before has left of all slices.
//   counts [pairs][slices][kPasses][kBins], above [pairs][slices][kPasses] (tokens of the slices in front that rank above by a pass's digit),
//   found [pairs][kPasses]
template <int PASS>  // kPasses: the places
__global__ __launch_bounds__(kSelectThreads) void paged_select_slices_kernel(const EvictArgs a, unsigned* all_counts, unsigned* all_above, Found* all_found) {
  __shared__ unsigned counts[kBins];
  __shared__ unsigned shared[kSelectThreads / 64 + 2];
  const int slice = blockIdx.x, slices = gridDim.x, head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, hi = kBins - 1 - 2 * tid;
  const int lane = tid & 63, wave = tid >> 6;
  const int64_t pair = (int64_t)b * a.kv_heads + head;
  Selection x = selection_of(a, head, b, slice, slices);
  if (PASS == 0 && slice == 0) place_ends(a, x);
  if (x.len <= a.budget || x.wanted == 0) return;
  unsigned* pair_counts = all_counts + pair * slices * (kPasses * kBins);
  unsigned* pair_above = all_above + pair * slices * kPasses;
  auto counts_of = [&](int s, int pass) { return (const uint2*)(pair_counts + (s * kPasses + pass) * kBins + hi - 1); };  // .y: the higher value
  auto sum_of = [&](unsigned v) {  // over the workgroup
    const unsigned w = (unsigned)wave_sum((int)v);
    if (lane == 0) shared[wave] = w;
    __syncthreads();
    unsigned t = 0;
    for (int i = 0; i < kSelectThreads / 64; ++i) t += shared[i];
    __syncthreads();
    return t;
  };
  Found f{0, x.wanted};
  if constexpr (PASS > 1) f = all_found[pair * kPasses + PASS - 2];
  unsigned above = 0, equal = 0;  // in the slices in front: by the digit just found, tokens that rank above, those that rank the same
  if constexpr (PASS > 0) {
    unsigned c0 = 0, c1 = 0, front0 = 0, front1 = 0;
#pragma unroll 16
    for (int s = 0; s < slices; ++s) {
      const uint2 c = *counts_of(s, PASS - 1);
      front0 += s < slice ? c.y : 0;
      front1 += s < slice ? c.x : 0;
      c0 += c.y;
      c1 += c.x;
    }
    find_digit(c0, c1, PASS - 1, f, shared);
    const int digit = (int)(f.prefix >> digit_shift(PASS - 1) & ((1u << digit_bits(PASS - 1)) - 1));
    above = sum_of((hi > digit ? front0 : 0) + (hi - 1 > digit ? front1 : 0));
    equal = (hi == digit ? front0 : 0) + (hi - 1 == digit ? front1 : 0);
  }
  if constexpr (PASS < kPasses) {
    if constexpr (PASS > 0) {
      if (tid == 0) {
        pair_above[slice * kPasses + PASS - 1] = above;
        if (slice == 0) all_found[pair * kPasses + PASS - 1] = f;
      }
    }
    count_digits(a, x.table, head, x.s, true, PASS, f.prefix, counts);
    unsigned* to = pair_counts + (slice * kPasses + PASS) * kBins;
    for (int i = tid; i < kBins; i += kSelectThreads) to[i] = counts[i];
  } else {
    for (int pass = 0; pass < kPasses - 1; ++pass) above += pair_above[slice * kPasses + pass];
    equal = sum_of(equal);
    place_tokens(a, x.table, head, x.s, true, x.kept, a.first + (int)above + min((int)equal, (int)f.wanted), (int)equal, f, counts);
  }
}

// Where only tokens whose page is there are to stay: the others out of the list, which is as long for all KV heads, since they rank below everything.
// A thread a place, 1024 at a time, and written no further than it has been read.  (Two dependent reads a turn, some 0.9 us: 16 sequences of 7.5 K
// tokens to 4 K, 8 KV heads, take 4 us more by it, one of 128 K to 32 K, 4 KV heads, 29.)
__global__ __launch_bounds__(kSelectThreads) void paged_present_kernel(const EvictArgs a) {
  __shared__ int counts[2][kSelectThreads / 64];  // in turn, so that one barrier each suffices
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* kept = a.kept + ((int64_t)b * a.kv_heads + head) * a.budget;
  const int* table = a.c.table + b * a.c.table_stride;
  int placed = 0;
  for (int j0 = 0, turn = 0; j0 < a.budget; j0 += kSelectThreads, turn ^= 1) {
    const int key = j0 + tid < a.budget ? kept[j0 + tid] : -1;
    const bool there = key >= 0 && (unsigned)table[key >> a.c.page_shift] < (unsigned)a.c.pages;
    const uint64_t mine = __builtin_amdgcn_ballot_w64(there);
    if (lane == 0) counts[turn][wave] = __builtin_popcountll(mine);
    __syncthreads();
    int front = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kSelectThreads / 64; ++i) {
      front += i < wave ? counts[turn][i] : 0;
      all += counts[turn][i];
    }
    if (there) kept[placed + front + __builtin_popcountll(mine & (((uint64_t)1 << lane) - 1))] = key;
    placed += all;
  }
  for (int j = placed + tid; j < a.budget; j += kSelectThreads) kept[j] = -1;
  if (head == 0 && tid == 0) a.kept_lens[b] = placed;  // (which may be the call's own lens: nothing here goes by those)
}

// 16 bytes a thread of a kept token's K and V.  The lengths are written here, not where tokens are selected: kept_lens may be the call's own lens,
// which every workgroup of a selection reads, and here one that has been written already says the same.
__global__ __launch_bounds__(256) void paged_move_kernel(const EvictArgs a, int row16) {
  const int head = blockIdx.y, b = blockIdx.z;
  const int rows = 256 / row16, c16 = threadIdx.x % row16;
  const int* kept = a.kept + ((int64_t)b * a.kv_heads + head) * a.budget;
  const int stay = a.present ? a.kept_lens[b] : min(clamped(a.c.lens[b], 0, a.c.table_pages << a.c.page_shift), a.budget);
  if (!a.present && head == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.kept_lens[b] = stay;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int mask = (1 << a.c.page_shift) - 1;
  for (int j = blockIdx.x * rows + threadIdx.x / row16; j < stay; j += gridDim.x * rows) {
    const int key = kept[j];
    const int page = a.c.table[b * a.c.table_stride + (key >> a.c.page_shift)];
    const int page_to = a.kept_table[b * a.kept_stride + (j >> a.c.page_shift)];
    if ((unsigned)page >= (unsigned)a.c.pages || (unsigned)page_to >= (unsigned)a.c.pages) continue;
    const int64_t from = page_row(a.c, page, head, key) + c16 * 16, to = page_row(a.c, page_to, head, j) + c16 * 16;
    const u32x4 x = *(const u32x4*)(a.c.k + from), y = *(const u32x4*)(a.c.v + from);
    *(u32x4*)(a.c.k + to) = x;
    *(u32x4*)(a.c.v + to) = y;
    if (c16 == 0)
      a.scores[(((int64_t)page_to * a.kv_heads + head) << a.c.page_shift) + (j & mask)] =
          a.scores[(((int64_t)page * a.kv_heads + head) << a.c.page_shift) + (key & mask)];
  }
}

hipError_t launch_paged_evict(const EvictArgs& a, int dim, hipStream_t stream) {
  if (a.c.batch <= 0 || a.kv_heads <= 0) return hipSuccess;
  if (a.kv_heads > 65535 || a.c.batch > 65535) return hipErrorInvalidValue;
  // Slices of as many tokens as a workgroup keeps the ranks of, for as long as that many workgroups find a compute unit and their counts
  // room in the workspace.  (One sequence of 128 K tokens, 4 KV heads, the move among it: 60 us; slices of half and twice that 65 and 73.)
  const int64_t pairs_ = (int64_t)a.c.batch * a.kv_heads, keys = (int64_t)a.c.table_pages << a.c.page_shift;
  const int64_t slice_bytes = kPasses * (kBins + 1) * sizeof(unsigned), pair_bytes = kPasses * sizeof(Found);
  const int64_t slice_tokens = kHeld * kSelectThreads;
  int64_t slices = (keys + slice_tokens - 1) / slice_tokens;
  slices = slices < 512 / pairs_ ? slices : 512 / pairs_;
  const int64_t room = (((int64_t)a.workspace_bytes - 8) / pairs_ - pair_bytes) / slice_bytes;
  slices = slices < room ? slices : room;
  if (slices < 2) {
    paged_select_kernel<<<dim3((unsigned)a.kv_heads, (unsigned)a.c.batch), kSelectThreads, 0, stream>>>(a);
  } else {
    unsigned* counts = (unsigned*)a.workspace;
    unsigned* above = counts + pairs_ * slices * kPasses * kBins;
    Found* found = (Found*)(above + ((pairs_ * slices * kPasses + 1) & ~(int64_t)1));
    const dim3 grid((unsigned)slices, (unsigned)a.kv_heads, (unsigned)a.c.batch);
    paged_select_slices_kernel<0><<<grid, kSelectThreads, 0, stream>>>(a, counts, above, found);
    paged_select_slices_kernel<1><<<grid, kSelectThreads, 0, stream>>>(a, counts, above, found);
    paged_select_slices_kernel<2><<<grid, kSelectThreads, 0, stream>>>(a, counts, above, found);
    paged_select_slices_kernel<3><<<grid, kSelectThreads, 0, stream>>>(a, counts, above, found);
  }
  if (a.present) paged_present_kernel<<<dim3((unsigned)a.kv_heads, (unsigned)a.c.batch), kSelectThreads, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int rows = 256 / (dim / 8);
  const int64_t pairs = (int64_t)a.c.batch * a.kv_heads, enough = (8192 + pairs - 1) / pairs;
  int64_t blocks = ((int64_t)a.budget + rows - 1) / rows;
  if (blocks > enough) blocks = enough;
  paged_move_kernel<<<dim3((unsigned)blocks, (unsigned)a.kv_heads, (unsigned)a.c.batch), 256, 0, stream>>>(a, dim / 8);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace ringattn
