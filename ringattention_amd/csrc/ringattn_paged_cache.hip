// gfx950 (CDNA4) kernels around the paged cache itself: new rows into it, the attention weight that its tokens have drawn, and the
// eviction that keeps those that drew most.
//
//   paged_append_kernel  : K and V rows of the new tokens to their places.  A copy: 16 bytes a thread.
//   paged_weights_kernel : score[key] += sum over queries of exp(scale q k - LSE).  The sum runs over queries where attention's runs
//       over keys, so a workgroup owns keys: K fragments stay in registers, the query rows pass by, S^T = K Q^T on MFMAs, and a
//       lane adds up the weights of its 16 keys over every 32nd query; lanes meet at the end.  One owner per score: no atomics, the
//       same bits in every run.
//   paged_select_kernel  : the places of a sequence's KV head that stay.  The budget-th largest score is found by its bits, from the
//       highest on, in counts of how many scores share the bits so far.
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
  // the sequence that token t is of: the last one that begins at or before it
  int lo = 0, hi = a.c.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.c.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int start = a.c.starts[lo], end = a.c.starts[lo + 1];
  if (t < start || t >= end) return;  // in front of the first, behind the last
  const int64_t key = (int64_t)a.c.lens[lo] - end + t;
  const int64_t entry = key >> a.c.page_shift;
  if (key < 0 || entry >= a.c.table_pages) return;
  const int page = a.c.table[lo * a.c.table_stride + entry];
  if ((unsigned)page >= (unsigned)a.c.pages) return;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int64_t from = t * a.ts + head * a.hs + c16 * 16, to = page_row(a.c, page, head, (int)key) + c16 * 16;
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
constexpr int kWeightWaves = 8, kWeightKeys = kWeightWaves * kKeyTile;

template <int DT, int D>
__global__ __launch_bounds__(64 * kWeightWaves) void paged_weights_kernel(const WeightsArgs a) {
  using E = Elem<DT>;
  constexpr int KS = D / 16;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.z, head = blockIdx.y;
  const Seq s = seq_of(a.c, b);
  if (s.n == 0) return;
  const int rows = s.n * a.group, before = s.len - s.n;
  constexpr float kLog2e = 1.4426950408889634f;
  for (int key0 = (blockIdx.x * kWeightWaves + wave) * kKeyTile; key0 < s.len; key0 += gridDim.x * kWeightKeys) {
    const int key = key0 + n, entry = key >> a.c.page_shift;
    int page = entry < a.c.table_pages && key < s.len ? a.c.table[b * a.c.table_stride + entry] : -1;
    if ((unsigned)page >= (unsigned)a.c.pages) page = -1;
    s16x8 kfr[KS];
    {
      const char* src = a.c.k + page_row(a.c, max(page, 0), head, key) + h * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kfr[ks] = *(const s16x8*)(src + ks * 32);
    }
    // the new tokens that see any of these keys
    int i0 = 0, i1 = s.n;
    if (a.causal) i0 = max(0, key0 - before);
    if (a.window > 0 && key0 >= a.sinks) i1 = min(s.n, key0 + kKeyTile - 1 + a.window - before);
    float w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = 0.f;
    for (int r0 = i0 * a.group; r0 < i1 * a.group; r0 += 32) {
      const int r = min(r0 + n, rows - 1), token = quotient(r, a.by_group), q_head = head * a.group + r - token * a.group;
      const char* qrow = a.q + (s.start + token) * a.q_ts + q_head * a.q_hs + h * 16;
      float lse = a.lse[(int64_t)q_head * a.c.tokens + s.start + token] * kLog2e;
      if (r0 + n >= rows || lse == -INFINITY) lse = INFINITY;  // no row, or one that saw nothing: weight 0
      f32x16 sacc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sacc[e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sacc = E::mma(kfr[ks], *(const s16x8*)(qrow + ks * 32), sacc);
      const int lim = a.causal ? min(s.len, before + token + 1) : s.len, low = a.window > 0 ? before + token - a.window : -1;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = key0 + 8 * (e >> 2) + (e & 3) + 4 * h;
        const bool hidden = k >= lim || (k <= low && k >= a.sinks) || lse == INFINITY;
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[e], a.scale_log2, -lse));
        w[e] += hidden ? 0.f : x;
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) w[e] += __shfl_xor(w[e], d);
    // lane (n, h) of n < 16 has the sum of accumulator n of half h
    float mine = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) mine = n == e ? w[e] : mine;
    const int k = key0 + 8 * (n >> 2) + (n & 3) + 4 * h;
    const int at = __shfl(page, (k - key0) & 31);
    if (n < 16 && at >= 0 && k < s.len) {
      float* to = a.scores + (((int64_t)at * a.kv_heads + head) << a.c.page_shift) + (k & ((1 << a.c.page_shift) - 1));
      *to += mine;
    }
  }
}

hipError_t launch_paged_weights(const WeightsArgs& a, int dtype, int dim, hipStream_t stream) {
  const int64_t keys = (int64_t)a.c.table_pages << a.c.page_shift;
  const int64_t pairs = (int64_t)a.c.batch * a.kv_heads;
  if (pairs <= 0 || keys <= 0) return hipSuccess;
  int64_t blocks = (keys + kWeightKeys - 1) / kWeightKeys;
  const int64_t enough = (4096 + pairs - 1) / pairs;
  if (blocks > enough) blocks = enough;
  if (a.kv_heads > 65535 || a.c.batch > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)a.kv_heads, (unsigned)a.c.batch);
  if (dtype == 0 && dim == 64) paged_weights_kernel<0, 64><<<grid, 64 * kWeightWaves, 0, stream>>>(a);
  else if (dtype == 1 && dim == 64) paged_weights_kernel<1, 64><<<grid, 64 * kWeightWaves, 0, stream>>>(a);
  else if (dtype == 0 && dim == 128) paged_weights_kernel<0, 128><<<grid, 64 * kWeightWaves, 0, stream>>>(a);
  else if (dtype == 1 && dim == 128) paged_weights_kernel<1, 128><<<grid, 64 * kWeightWaves, 0, stream>>>(a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

// ---- eviction ----------------------------------------------------------------------
// Larger scores have larger ranks; a NaN and a token whose page is not there rank with -inf.
static __device__ __forceinline__ unsigned rank_of(float x) {
  if (!(x == x)) x = -INFINITY;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);  // (-0 as 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kDigit = 11;

__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(const EvictArgs a) {
  __shared__ unsigned counts[1 << kDigit];
  __shared__ int wave_total[kSelectThreads / 64];
  __shared__ unsigned found_digit, found_above;
  const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = clamped(a.c.lens[b], 0, a.c.table_pages << a.c.page_shift);
  int* kept = a.kept + ((int64_t)b * a.kv_heads + head) * a.budget;
  const int stay = min(len, a.budget);
  if (head == 0 && tid == 0) a.kept_lens[b] = stay;
  for (int j = stay + tid; j < a.budget; j += kSelectThreads) kept[j] = -1;
  if (len <= a.budget) {
    for (int j = tid; j < len; j += kSelectThreads) kept[j] = j;
    return;
  }
  const int* table = a.c.table + b * a.c.table_stride;
  auto rank_at = [&](int key) {
    const int page = table[key >> a.c.page_shift];
    if ((unsigned)page >= (unsigned)a.c.pages) return rank_of(-INFINITY);
    return rank_of(a.scores[(((int64_t)page * a.kv_heads + head) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))]);
  };
  const int from = a.first, to = len - a.last;  // the tokens whose scores decide
  unsigned wanted = a.budget - a.first - a.last;  // of them, so many stay
  // the rank of the last one that stays, digit by digit: `prefix` so far, `wanted` of those that share it stay
  unsigned prefix = 0, known = 0;
  for (int shift = 32; wanted > 0 && shift > 0;) {
    const int bits = min(kDigit, shift);
    shift -= bits;
    for (int i = tid; i < 1 << kDigit; i += kSelectThreads) counts[i] = 0;
    __syncthreads();
    for (int key = from + tid; key < to; key += kSelectThreads) {
      const unsigned r = rank_at(key);
      if ((r & known) == prefix) atomicAdd(&counts[r >> shift & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // the digit at which the count from the top reaches `wanted`: a thread has two of them, the highest first
    const int hi = (1 << kDigit) - 1 - 2 * tid, c0 = (int)counts[hi], c1 = (int)counts[hi - 1];
    const int both = c0 + c1, upto = wave_scan(both, lane);
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    int above = upto - both;
    for (int w = 0; w < wave; ++w) above += wave_total[w];
    const int want = (int)wanted;
    if (above < want && want <= above + c0) {
      found_digit = hi;
      found_above = above;
    } else if (above + c0 < want && want <= above + both) {
      found_digit = hi - 1;
      found_above = above + c0;
    }
    __syncthreads();
    prefix |= found_digit << shift;
    known |= ((1u << bits) - 1) << shift;
    wanted -= found_above;
    __syncthreads();
  }
  // in order: what ranks above stays, and the first `wanted` of those that rank the same.  A wave has 64 tokens at a time, one wave's
  // after the other's.
  const bool any = a.budget > a.first + a.last;
  int placed = 0, equal_before = 0;
  for (int key0 = 0; key0 < len; key0 += kSelectThreads) {
    const int key = key0 + tid;
    bool more = false, same = false;
    if (key < len) {
      if (key < from || key >= to) more = true;
      else if (any) {
        const unsigned r = rank_at(key);
        more = r > prefix;
        same = r == prefix;
      }
    }
    const uint64_t sames = __builtin_amdgcn_ballot_w64(same);
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    if (lane == 0) wave_total[wave] = __builtin_popcountll(sames);
    __syncthreads();
    int eq = equal_before, eq_all = 0;
    for (int w = 0; w < kSelectThreads / 64; ++w) {
      if (w < wave) eq += wave_total[w];
      eq_all += wave_total[w];
    }
    equal_before += eq_all;
    const bool stays = more || (same && eq + __builtin_popcountll(sames & below) < (int)wanted);
    const uint64_t staying = __builtin_amdgcn_ballot_w64(stays);
    __syncthreads();
    if (lane == 0) wave_total[wave] = __builtin_popcountll(staying);
    __syncthreads();
    int at = placed, all = 0;
    for (int w = 0; w < kSelectThreads / 64; ++w) {
      if (w < wave) at += wave_total[w];
      all += wave_total[w];
    }
    placed += all;
    at += __builtin_popcountll(staying & below);
    if (stays && at < a.budget) kept[at] = key;
    __syncthreads();
  }
}

// 16 bytes a thread of a kept token's K and V.
__global__ __launch_bounds__(256) void paged_move_kernel(const EvictArgs a, int row16) {
  const int head = blockIdx.y, b = blockIdx.z;
  const int rows = 256 / row16, c16 = threadIdx.x % row16;
  const int* kept = a.kept + ((int64_t)b * a.kv_heads + head) * a.budget;
  const int len = clamped(a.c.lens[b], 0, a.c.table_pages << a.c.page_shift), stay = min(len, a.budget);
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
  paged_select_kernel<<<dim3((unsigned)a.kv_heads, (unsigned)a.c.batch), kSelectThreads, 0, stream>>>(a);
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
