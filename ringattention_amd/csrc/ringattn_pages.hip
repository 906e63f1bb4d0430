// gfx950 (CDNA4) kernels and host side: the pages of a cache (ringattn_pages_* in include/ringattn.h) -- which rows of the table share them, which
// are free, and the copies that follow.  Counts and places are whole numbers, taken in the order of rows and pages, so that every run gives the
// same table; what moves K and V is a copy.
//
//   pages_share_kernel   : rows of the table become what they keep of their parents'; counts of the pages follow (additions to
//       integers: in any order the same).
//   pages_grow_kernel    : how many pages every row wants, and the first free ones to them, in the order of the rows.  One workgroup: a step of a serving
//       loop wants a page for every so-many-th row, and finds them in front.
//   pages_settle_kernel  : rows that others were made of come to the table; shared pages that are written on are copied.
//   pages_count_kernel, pages_rank_kernel, pages_move_kernel : compaction.  Of n pages in use, those from place n on go to the free ones in front of
//       it, the i-th to the i-th.
#include "ringattn.h"
#include "ringattn_paged.h"

#include <cstring>

namespace ringattn {
namespace pages {

using paged::clamped;
using paged::wave_scan;
using paged::wave_sum;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxRows = 4096, kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBlock = 4096;        // pages that a workgroup of the compaction looks at
constexpr int kOwnCounts = 8;       // up to so many blocks, every workgroup counts all pages itself
constexpr int kUnits = 1024;        // 16-byte units of a page's K, and of its V, that a workgroup copies

// A pool of pages, rows of dim 16-bit values.
struct Pool {
  char *k, *v;
  float* scores;                     // [pages, kv_heads, page] or NULL
  int64_t page_stride, head_stride;  // bytes
  int token_stride;
  int kv_heads, page_shift, unit_shift;  // 2^unit_shift units of 16 bytes a row
  __device__ __forceinline__ int64_t units() const { return (int64_t)kv_heads << (page_shift + unit_shift); }
  __device__ __forceinline__ int64_t place(int page, int64_t unit) const {
    const int token = (int)(unit >> unit_shift) & ((1 << page_shift) - 1);
    return page * page_stride + (unit >> (unit_shift + page_shift)) * head_stride + (int64_t)token * token_stride + ((unit & ((1 << unit_shift) - 1)) << 4);
  }
};
// Units [first, first + kUnits) of a page, and the scores that go with them, by 256 threads.
static __device__ __forceinline__ void copy_units(const Pool& from, const Pool& to, int source, int target, int64_t first) {
  constexpr int EACH = kUnits / 256;
  const int64_t units = from.units();
  u32x4 k[EACH], v[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t u = min(first + i * 256 + (int64_t)threadIdx.x, units - 1), at = from.place(source, u);
    k[i] = *(const u32x4*)(from.k + at);
    v[i] = *(const u32x4*)(from.v + at);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t u = first + i * 256 + threadIdx.x;
    if (u >= units) break;
    const int64_t at = to.place(target, u);
    *(u32x4*)(to.k + at) = k[i];
    *(u32x4*)(to.v + at) = v[i];
  }
  if (from.scores && to.scores) {
    const int64_t rows = units >> from.unit_shift;
    for (int64_t r = (first >> from.unit_shift) + threadIdx.x; r < min(rows, (first + kUnits) >> from.unit_shift); r += 256)
      to.scores[target * rows + r] = from.scores[source * rows + r];
  }
}

struct Args {
  int* refs;
  int* table;
  int* lens;
  int64_t table_stride;
  int pages, rows, table_pages, page_shift;
  const int* parents;  // [rows] or NULL
  const int* add;      // [rows] or NULL
  int* missing;        // [rows] or NULL
  int2* pairs;         // copies of an update [rows], moves of a compaction [pages]: from, to, or -1; or NULL
  // scratch
  int* made;           // [rows, table_pages]: rows that others were made of
  int2* told;          // [rows]: where the row's entries of `made` begin and end; of a compaction [0]: pages in use, and how many move
  int2* copies;        // [rows]: pages that are copied, from, to; [0, copied[0])
  int* copied;         // [1]
  int* list;           // [pages]: free pages; of a compaction: pages that move
  int* slots;          // [pages]: where they go
  int* counts;         // [pages / kBlock + 1] pages in use
  int* used;           // compaction: [1]
  int* moved;          // [pages] or NULL
};

// What a row is to become.
struct Row {
  int parent;     // its own number; another row's; -1: it begins anew
  int had, want;  // tokens that it begins with, and that it is to have (may pass what the table has room for)
  int kept;       // entries that it begins with
  int old;        // entries that it had
  __device__ __forceinline__ Row(const Args& a, int b) {
    const int room = a.table_pages << a.page_shift, page = 1 << a.page_shift;
    parent = a.parents ? a.parents[b] : b;
    if ((unsigned)parent >= (unsigned)a.rows) parent = -1;
    had = parent < 0 ? 0 : clamped(a.lens[parent], 0, room);
    const int64_t sum = (int64_t)had + (a.add ? a.add[b] : 0);
    want = (int)(sum < 0 ? 0 : sum > INT32_MAX ? INT32_MAX : sum);
    kept = (min(had, want) + page - 1) >> a.page_shift;
    old = (clamped(a.lens[b], 0, room) + page - 1) >> a.page_shift;
  }
};

__global__ __launch_bounds__(256) void pages_share_kernel(const Args a) {
  const int b = blockIdx.x;
  const Row r(a, b);
  const bool itself = r.parent == b;
  int* const row = a.table + b * a.table_stride;
  const int* const from = r.parent < 0 ? row : a.table + r.parent * a.table_stride;
  auto count = [&](int page, int by) {
    if ((unsigned)page < (unsigned)a.pages) atomicAdd(a.refs + page, by);
  };
  const int begin = itself ? r.kept : 0, end = max(r.kept, r.old);
  for (int e = begin + (int)(blockIdx.y * 256 + threadIdx.x); e < end; e += gridDim.y * 256) {
    if (e < r.old) count(row[e], -1);
    if (itself) {  // (rows that are made of this one read what they keep of it from the table as it was)
      if (!a.parents) row[e] = -1;
      else a.made[(int64_t)b * a.table_pages + e] = -1;
    } else {
      const int page = e < r.kept ? from[e] : -1;
      count(page, 1);
      a.made[(int64_t)b * a.table_pages + e] = page;
    }
  }
}

// Inclusive sums over a workgroup of kThreads; `all`: of all of them.  Two barriers.
static __device__ __forceinline__ int scan_all(int x, int* sums, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_scan(x);
  __syncthreads();
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  const int s = wave_scan(lane < kWaves ? sums[lane] : 0);
  all = __builtin_amdgcn_readlane(s, kWaves - 1);
  return upto + (wave > 0 ? __builtin_amdgcn_readlane(s, __builtin_amdgcn_readfirstlane(wave) - 1) : 0);
}

// Four pages' counts; of pages behind the last, `none`.
static __device__ __forceinline__ i32x4 counts_of(const Args& a, int64_t page, int none) {
  if (page + 3 < a.pages) return *(const i32x4*)(a.refs + page);
  i32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = page + i < a.pages ? a.refs[page + i] : none;
  return x;
}

__global__ __launch_bounds__(kThreads) void pages_grow_kernel(const Args a) {
  constexpr int EACH = kMaxRows / kThreads;
  __shared__ int upto[kMaxRows], first[kMaxRows], sums[4][kWaves];
  const int tid = threadIdx.x, room = a.table_pages << a.page_shift, page = 1 << a.page_shift;
  // rows 4 tid to 4 tid + 3
  int had[EACH], want[EACH], need[EACH], kept[EACH], torn[EACH], old[EACH];
  bool itself[EACH];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int b = EACH * tid + i;
    need[i] = had[i] = want[i] = kept[i] = old[i] = 0;
    torn[i] = -1;
    itself[i] = true;
    if (b >= a.rows) continue;
    const Row r(a, b);
    had[i] = r.had;
    want[i] = r.want;
    kept[i] = r.kept;
    old[i] = r.old;
    itself[i] = r.parent == b;
    if (r.want <= r.had || r.want > room) continue;
    if (r.had & (page - 1)) {  // the last entry that it keeps is written on: copied, if it is not the row's alone
      const int e = r.had >> a.page_shift, x = itself[i] ? a.table[b * a.table_stride + e] : a.made[(int64_t)b * a.table_pages + e];
      if ((unsigned)x < (unsigned)a.pages && a.refs[x] > 1) torn[i] = x;
    }
    need[i] = ((r.want - 1) >> a.page_shift) + 1 - r.kept + (torn[i] >= 0 ? 1 : 0);
    mine += need[i];
  }
  int total, before = scan_all(mine, sums[0], total) - mine;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    before += need[i];
    upto[EACH * tid + i] = before;
    first[EACH * tid + i] = kept[i] - (torn[i] >= 0 ? 1 : 0);
  }
  // the first `total` free pages, 16 K of them looked at at a time
  int found = 0;
  __syncthreads();
  for (int64_t base = 0; base < a.pages && found < total; base += 4 * 4 * kThreads) {
    i32x4 x[4];
    int n[4], at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = counts_of(a, base + (u * kThreads + tid) * 4, 1);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      n[u] = (x[u][0] == 0) + (x[u][1] == 0) + (x[u][2] == 0) + (x[u][3] == 0);
      at[u] = wave_scan(n[u]);
      if ((tid & 63) == 63) sums[u][tid >> 6] = at[u];
    }
    __syncthreads();
    // 4 x 16 sums of waves, a lane each
    const int lane = tid & 63, s = wave_scan((&sums[0][0])[lane]), all = __builtin_amdgcn_readlane(s, 63);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = u * kWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
      int rank = found + at[u] - n[u] + (w > 0 ? __builtin_amdgcn_readlane(s, w - 1) : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (x[u][i] == 0) {
          if (rank < total) a.list[rank] = (int)(base + (u * kThreads + tid) * 4 + i);
          ++rank;
        }
    }
    found += all;
  }
  found = min(found, total);
  __syncthreads();  // (all waves see the list and the rows of this workgroup's own)
  // all lengths have been read: they may be written
  int copies = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int b = EACH * tid + i;
    if (b >= a.rows) continue;
    const bool grows = want[i] > had[i], granted = grows && want[i] <= room && upto[b] <= found;
    const int now = grows && !granted ? had[i] : want[i];
    a.lens[b] = now;
    if (a.missing) a.missing[b] = grows && !granted;
    int2 copy{-1, -1};
    if (granted && torn[i] >= 0) {
      copy = int2{torn[i], a.list[upto[b] - need[i]]};
      atomicAdd(a.refs + torn[i], -1);
      ++copies;
    }
    torn[i] = copy.x;
    if (a.pairs) a.pairs[b] = copy;
    if (a.parents) a.told[b] = int2{itself[i] ? kept[i] - (copy.x >= 0 ? 1 : 0) : 0, max((now + page - 1) >> a.page_shift, old[i])};
    if (!granted) first[b] = -1;
  }
  int all_copies, at_copy = scan_all(copies, sums[0], all_copies) - copies;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (torn[i] >= 0) a.copies[at_copy++] = int2{torn[i], a.list[upto[EACH * tid + i] - need[i]]};
  if (tid == 0) a.copied[0] = all_copies;
  for (int j = tid; j < found; j += kThreads) {
    int lo = 0, hi = kMaxRows - 1;  // the first row whose pages end behind j
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (upto[mid] > j) hi = mid;
      else lo = mid + 1;
    }
    if (first[lo] < 0) continue;
    const int begin = lo > 0 ? upto[lo - 1] : 0, e = first[lo] + j - begin, x = a.list[j];
    a.refs[x] = 1;
    if (a.parents) a.made[(int64_t)lo * a.table_pages + e] = x;
    else a.table[lo * a.table_stride + e] = x;
  }
}

// Workgroups [0, entry_blocks): entries of the table, with parents.  The others: pages, piece by piece.
__global__ __launch_bounds__(256) void pages_settle_kernel(const Args a, const Pool pool, int pieces, int entry_blocks, int each) {
  if ((int)blockIdx.x < entry_blocks) {
    const int b = blockIdx.x / each;
    const int2 t = a.told[b];
    for (int e = t.x + (int)((blockIdx.x - b * each) * 256 + threadIdx.x); e < t.y; e += each * 256)
      a.table[b * a.table_stride + e] = a.made[(int64_t)b * a.table_pages + e];
    return;
  }
  const int64_t items = (int64_t)a.copied[0] * pieces;
  for (int64_t i = blockIdx.x - entry_blocks; i < items; i += gridDim.x - entry_blocks) {
    const int64_t j = i / pieces;
    const int2 copy = a.copies[j];
    copy_units(pool, pool, copy.x, copy.y, (i - j * pieces) * kUnits);
  }
}

// ---- compaction
__global__ __launch_bounds__(256) void pages_count_kernel(const Args a) {
  __shared__ int sums[4];
  int n = 0;
#pragma unroll
  for (int u = 0; u < kBlock / 1024; ++u) {
    const i32x4 x = counts_of(a, (int64_t)blockIdx.x * kBlock + (u * 256 + (int)threadIdx.x) * 4, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) n += x[i] != 0;
  }
  const int all = wave_sum(n);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = all;
  __syncthreads();
  if (threadIdx.x == 0) a.counts[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// A workgroup's pages: how many in use lie in front of each, and with that its place in one of the two lists.  Every workgroup works out for
// itself how many there are in all (n), and how many in front of place n.  OWN: from the pages themselves, up to
// kOwnCounts blocks of them, which is a launch less.  (1128 pages of 2821 compacted: 82.0 us, 83.6 with the launch.)
template <bool OWN> __global__ __launch_bounds__(kThreads) void pages_rank_kernel(const Args a) {
  __shared__ int sums[kWaves], own[OWN ? kOwnCounts : 1], parts[OWN ? kOwnCounts : 1][kWaves];
  static_assert(kBlock == 4 * kThreads, "four pages a thread");
  const int tid = threadIdx.x, blocks = gridDim.x;
  const int* counts = a.counts;
  if constexpr (OWN) {
    i32x4 x[kOwnCounts];
#pragma unroll
    for (int i = 0; i < kOwnCounts; ++i) x[i] = i < blocks ? counts_of(a, (int64_t)i * kBlock + 4 * tid, 0) : i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kOwnCounts; ++i) {
      const int all = wave_sum((x[i][0] != 0) + (x[i][1] != 0) + (x[i][2] != 0) + (x[i][3] != 0));
      if ((tid & 63) == 0) parts[i][tid >> 6] = all;
    }
    __syncthreads();
    if (tid < kOwnCounts) {
      int all = 0;
      for (int w = 0; w < kWaves; ++w) all += parts[tid][w];
      own[tid] = all;
    }
    __syncthreads();
    counts = own;
  }
  int all = 0, front = 0;
  for (int i = tid; i < blocks; i += kThreads) {
    all += counts[i];
    front += i < (int)blockIdx.x ? counts[i] : 0;
  }
  int n, before;
  scan_all(all, sums, n);
  scan_all(front, sums, before);
  auto used_of = [&](int64_t page, int from, int& upto, i32x4& x) {  // pages in use in front of a thread's four
    x = counts_of(a, page, 0);
    const int mine = (x[0] != 0) + (x[1] != 0) + (x[2] != 0) + (x[3] != 0);
    int unused;
    upto = from + scan_all(mine, sums, unused) - mine;
  };
  // in front of place n: those of whole blocks, and of the block that n lies in
  int low = 0;
  for (int i = tid; i < blocks; i += kThreads) low += i < n / kBlock ? counts[i] : 0;
  int within = 0;
  {
    const int64_t page = (int64_t)(n / kBlock) * kBlock + 4 * tid;  // (behind the last where all are in use)
    const i32x4 x = counts_of(a, page, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) within += page + i < n && x[i] != 0;
  }
  int in_front;
  scan_all(low + within, sums, in_front);
  const int64_t page = (int64_t)blockIdx.x * kBlock + 4 * tid;
  int upto;
  i32x4 x;
  used_of(page, before, upto, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = (int)page + i;
    if (page + i >= a.pages) break;
    const bool used = x[i] != 0;
    if (used && p >= n) a.list[upto - in_front] = p;
    if (!used && p < n) a.slots[p - upto] = p;
    if (a.moved && (!used || p < n)) a.moved[p] = used ? p : -1;
    upto += used;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.used[0] = n;
    a.told[0] = int2{n, n - in_front};  // for the next launch
  }
}

// Workgroups [0, table_blocks): entries of the table.  The others: pages, piece by piece (one piece that copies nothing where the caller does that).
__global__ __launch_bounds__(256) void pages_move_kernel(const Args a, const Pool pool, int pieces, int table_blocks) {
  const int2 t = a.told[0];
  const int n = t.x, m = t.y;
  if ((int)blockIdx.x < table_blocks) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; a.pairs && i < a.pages; i += (int64_t)table_blocks * 256)
      a.pairs[i] = i < m ? int2{a.list[i], a.slots[i]} : int2{-1, -1};
    if (m == 0) return;
    const int64_t entries = (int64_t)a.rows * a.table_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)table_blocks * 256) {
      const int64_t b = i / a.table_pages;
      int* const entry = a.table + b * a.table_stride + (i - b * a.table_pages);
      const int x = *entry;
      if (x < n || x >= a.pages) continue;
      int lo = 0, hi = m;  // the pages that move are in their order
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.list[mid] <= x) lo = mid;
        else hi = mid;
      }
      if (a.list[lo] == x) *entry = a.slots[lo];
    }
    return;
  }
  for (int64_t i = blockIdx.x - table_blocks; i < (int64_t)m * pieces; i += gridDim.x - table_blocks) {
    const int j = (int)(i / pieces), piece = (int)(i - (int64_t)j * pieces), from = a.list[j], to = a.slots[j];
    if (piece == 0 && threadIdx.x == 0) {
      a.refs[to] = a.refs[from];
      a.refs[from] = 0;
      if (a.moved) a.moved[from] = to;
    }
    if (pool.k) copy_units(pool, pool, from, to, (int64_t)piece * kUnits);
  }
}

// ---- pages from one pool to another
__global__ __launch_bounds__(256) void pages_copy_kernel(const Pool from, const Pool to, int from_pages, int to_pages, const int* pairs, int64_t items, int pieces) {
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t j = i / pieces;
    const int source = pairs[2 * j], target = pairs[2 * j + 1];
    if ((unsigned)source >= (unsigned)from_pages || (unsigned)target >= (unsigned)to_pages) continue;
    copy_units(from, to, source, target, (i - j * pieces) * kUnits);
  }
}

namespace {

inline bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
#define PG_CHECK(expr)                        \
  do {                                        \
    const int rc__ = (expr);                  \
    if (rc__ != RINGATTN_OK) return rc__;     \
  } while (0)

// Scratch: told, then the lists, then rows that others were made of.
struct Scratch {
  size_t told, copies, copied, list, slots, counts, made, bytes;
};
bool sizes_ok(int pages, int rows, int table_pages, int page_size) {
  return pages >= 1 && rows >= 1 && rows <= kMaxRows && table_pages >= 1 && page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0 &&
         (int64_t)table_pages * page_size <= (int64_t)1 << 30 && (int64_t)rows * table_pages <= (int64_t)1 << 30;
}
Scratch scratch_of(int pages, int rows, int table_pages) {
  Scratch s;
  auto up = [](size_t x) { return (x + 15) & ~(size_t)15; };
  s.told = 0;
  s.copies = s.told + up((size_t)rows * sizeof(int2));
  s.copied = s.copies + up((size_t)rows * sizeof(int2));
  s.list = s.copied + up(sizeof(int));
  s.slots = s.list + up((size_t)pages * sizeof(int));
  s.counts = s.slots + up((size_t)pages * sizeof(int));
  s.made = s.counts + up(((size_t)pages / kBlock + 1) * sizeof(int));
  s.bytes = s.made + up((size_t)rows * table_pages * sizeof(int));
  return s;
}

int check_pool(const ringattn_paged_pool* p, int pages, int page_size, Pool* out) {
  if (!p || !p->k || !p->v) return RINGATTN_ERR_NULL;
  if (p->dim != 64 && p->dim != 128) return RINGATTN_ERR_DIM;
  if (p->kv_heads < 1 || p->kv_heads > 65535) return RINGATTN_ERR_SHAPE;
  const int64_t most = (int64_t)1 << 40;
  if (p->token_stride < p->dim || p->token_stride > 1 << 24 || p->page_stride < p->dim || p->page_stride > most / 2 || p->head_stride < p->dim || p->head_stride > most)
    return RINGATTN_ERR_SHAPE;
  if ((double)pages * (double)p->page_stride > (double)((int64_t)1 << 60)) return RINGATTN_ERR_SHAPE;
  if ((p->token_stride | p->page_stride | p->head_stride) & 7) return RINGATTN_ERR_ALIGN;
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->scores, 4)) return RINGATTN_ERR_ALIGN;
  std::memset(out, 0, sizeof(*out));
  out->k = (char*)p->k;
  out->v = (char*)p->v;
  out->scores = p->scores;
  out->page_stride = p->page_stride * 2;
  out->head_stride = p->head_stride * 2;
  out->token_stride = (int)(p->token_stride * 2);
  out->kv_heads = p->kv_heads;
  out->page_shift = __builtin_ctz((unsigned)page_size);
  out->unit_shift = p->dim == 64 ? 3 : 4;
  return RINGATTN_OK;
}
// A pool, or none: then the caller makes the copies, for which it needs the pairs.
int check_pool_or_pairs(const ringattn_paged_pool* p, const ringattn_pages* pages, const int* pairs, Pool* out) {
  if (!aligned(pairs, 8)) return RINGATTN_ERR_ALIGN;
  std::memset(out, 0, sizeof(*out));
  if (!p) return pairs ? RINGATTN_OK : RINGATTN_ERR_NULL;
  return check_pool(p, pages->pages, pages->page_size, out);
}
int pieces_of(const Pool& p) { return (int)((((int64_t)p.kv_heads << (p.page_shift + p.unit_shift)) + kUnits - 1) / kUnits); }

int check_pages(const ringattn_pages* p, Args* a) {
  if (!p) return RINGATTN_ERR_NULL;
  if (!p->refs || !p->page_table || !p->lens) return RINGATTN_ERR_NULL;
  if (!sizes_ok(p->pages, p->rows, p->table_pages, p->page_size)) return RINGATTN_ERR_SHAPE;
  if (p->table_stride < p->table_pages || p->table_stride > (int64_t)1 << 40) return RINGATTN_ERR_SHAPE;
  if (!aligned(p->refs, 16) || !aligned(p->page_table, 4) || !aligned(p->lens, 4)) return RINGATTN_ERR_ALIGN;
  const Scratch s = scratch_of(p->pages, p->rows, p->table_pages);
  if (!p->scratch || p->scratch_bytes < s.bytes) return RINGATTN_ERR_WORKSPACE;
  if (!aligned(p->scratch, 16)) return RINGATTN_ERR_ALIGN;
  std::memset(a, 0, sizeof(*a));
  a->refs = p->refs;
  a->table = p->page_table;
  a->lens = p->lens;
  a->table_stride = p->table_stride;
  a->pages = p->pages;
  a->rows = p->rows;
  a->table_pages = p->table_pages;
  a->page_shift = __builtin_ctz((unsigned)p->page_size);
  char* w = (char*)p->scratch;
  a->told = (int2*)(w + s.told);
  a->copies = (int2*)(w + s.copies);
  a->copied = (int*)(w + s.copied);
  a->list = (int*)(w + s.list);
  a->slots = (int*)(w + s.slots);
  a->counts = (int*)(w + s.counts);
  a->made = (int*)(w + s.made);
  return RINGATTN_OK;
}
int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RINGATTN_OK : hip_failed(e);
}

}  // namespace

}  // namespace pages
}  // namespace ringattn

namespace pg = ringattn::pages;

extern "C" {

size_t ringattn_pages_scratch_bytes(int pages, int rows, int table_pages) {
  return pg::sizes_ok(pages, rows, table_pages, 16) ? pg::scratch_of(pages, rows, table_pages).bytes : 0;
}

int ringattn_pages_update(const ringattn_pages* pages, const ringattn_paged_pool* pool, const int* parents, const int* add, int* missing, int* copies,
                          void* stream_) {
  pg::Args a;
  pg::Pool p;
  PG_CHECK(pg::check_pages(pages, &a));
  PG_CHECK(pg::check_pool_or_pairs(pool, pages, copies, &p));
  if (!pg::aligned(parents, 4) || !pg::aligned(add, 4) || !pg::aligned(missing, 4)) return RINGATTN_ERR_ALIGN;
  a.parents = parents;
  a.add = add;
  a.missing = missing;
  a.pairs = (int2*)copies;
  hipStream_t stream = (hipStream_t)stream_;
  // workgroups of a row: all of its entries, 256 at a time, but no more than 4096 workgroups in all
  int each = (a.table_pages + 255) / 256;
  const int most = 4096 / a.rows > 1 ? 4096 / a.rows : 1;
  each = each < most ? each : most;
  const int pieces = pool ? pg::pieces_of(p) : 0, entry_blocks = parents ? a.rows * each : 0;
  const int64_t items = (int64_t)a.rows * pieces, copy_blocks = items < 4096 ? items : 4096;  // (a copy for every row at most)
  pg::pages_share_kernel<<<dim3((unsigned)a.rows, (unsigned)each), 256, 0, stream>>>(a);
  pg::pages_grow_kernel<<<1, pg::kThreads, 0, stream>>>(a);
  if (entry_blocks + copy_blocks > 0) pg::pages_settle_kernel<<<(unsigned)(entry_blocks + copy_blocks), 256, 0, stream>>>(a, p, pieces, entry_blocks, each);
  return pg::launched();
}

int ringattn_pages_compact(const ringattn_pages* pages, const ringattn_paged_pool* pool, int* used, int* moved, int* moves, void* stream_) {
  pg::Args a;
  pg::Pool p;
  PG_CHECK(pg::check_pages(pages, &a));
  PG_CHECK(pg::check_pool_or_pairs(pool, pages, moves, &p));
  if (!used) return RINGATTN_ERR_NULL;
  if (!pg::aligned(used, 4) || !pg::aligned(moved, 4)) return RINGATTN_ERR_ALIGN;
  a.used = used;
  a.moved = moved;
  a.pairs = (int2*)moves;
  hipStream_t stream = (hipStream_t)stream_;
  const unsigned blocks = (unsigned)((a.pages + (int64_t)pg::kBlock - 1) / pg::kBlock);
  const int64_t entries = ((int64_t)a.rows * a.table_pages + 1023) / 1024;
  const int table_blocks = (int)(entries < 512 ? entries : 512), pieces = pool ? pg::pieces_of(p) : 1;
  const int64_t items = (int64_t)(a.pages / 2) * pieces, move_blocks = items < 4096 ? items : 4096;  // (no more than half of the pages move)
  if (blocks <= (unsigned)pg::kOwnCounts) {
    pg::pages_rank_kernel<true><<<blocks, pg::kThreads, 0, stream>>>(a);
  } else {
    pg::pages_count_kernel<<<blocks, 256, 0, stream>>>(a);
    pg::pages_rank_kernel<false><<<blocks, pg::kThreads, 0, stream>>>(a);
  }
  pg::pages_move_kernel<<<(unsigned)(table_blocks + move_blocks), 256, 0, stream>>>(a, p, pieces, table_blocks);
  return pg::launched();
}

int ringattn_pages_copy(const ringattn_paged_pool* from, int from_pages, const ringattn_paged_pool* to, int to_pages, int page_size, const int* pairs, int n,
                        void* stream) {
  pg::Pool f, t;
  if (from_pages < 1 || to_pages < 1 || n < 0 || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) return RINGATTN_ERR_SHAPE;
  PG_CHECK(pg::check_pool(from, from_pages, page_size, &f));
  PG_CHECK(pg::check_pool(to, to_pages, page_size, &t));
  if (from->dim != to->dim || from->kv_heads != to->kv_heads || (from->scores == nullptr) != (to->scores == nullptr)) return RINGATTN_ERR_SHAPE;
  if (!pairs) return RINGATTN_ERR_NULL;
  if (!pg::aligned(pairs, 4)) return RINGATTN_ERR_ALIGN;
  if (n == 0) return RINGATTN_OK;
  const int pieces = pg::pieces_of(f);
  const int64_t items = (int64_t)n * pieces;
  pg::pages_copy_kernel<<<(unsigned)(items < 8192 ? items : 8192), 256, 0, (hipStream_t)stream>>>(f, t, from_pages, to_pages, pairs, items, pieces);
  return pg::launched();
}

}  // extern "C"
