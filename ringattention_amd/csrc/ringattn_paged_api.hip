// Host side of the paged cache's entry points (include/ringattn.h): checks, plan lifetime, launches.  Whatever the device arrays
// hold is the kernels' to check; everything that the host can see is checked here, before the first HIP call.
#include "ringattn.h"
#include "ringattn_paged.h"

#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <unordered_set>

namespace rp = ringattn::paged;

struct ringattn_paged_plan {
  ringattn_paged_params p;
  int kv_heads;
  float scale;
  int page_shift;
  void* ws = nullptr;
  bool own_ws = false;
};

namespace {

std::mutex g_paged_mu;
std::unordered_set<const void*> g_paged_plans;

inline bool plan_ok(const ringattn_paged_plan* pl) {
  std::lock_guard<std::mutex> lk(g_paged_mu);
  return pl && g_paged_plans.count(pl) != 0;
}
inline bool aligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// Rows of a KV head up to which a sequence has few: where a call is made of single tokens, or of some at a time, all of them, so that no
// workgroup has to find out that there are no others, and nothing is launched for those.
int few_most(int tokens, int batch, int most) { return batch > 1 && tokens < (int64_t)4 * batch ? INT32_MAX : most; }

int validate(const ringattn_paged_params* p) {
  if (!p) return RINGATTN_ERR_NULL;
  if (p->dim != 64 && p->dim != 128) return RINGATTN_ERR_DIM;
  if (p->dtype != RINGATTN_DTYPE_FP16 && p->dtype != RINGATTN_DTYPE_BF16) return RINGATTN_ERR_DTYPE;
  if (p->heads < 1 || p->kv_heads < 0 || (p->kv_heads > 0 && p->heads % p->kv_heads != 0)) return RINGATTN_ERR_SHAPE;
  if (p->heads > 65535) return RINGATTN_ERR_SHAPE;
  if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)) != 0) return RINGATTN_ERR_SHAPE;
  if (p->max_batch < 1 || p->max_batch > rp::kMaxBatch) return RINGATTN_ERR_SHAPE;
  if (p->max_tokens < 1 || (int64_t)p->max_tokens * p->heads > (int64_t)1 << 30) return RINGATTN_ERR_SHAPE;
  if (p->window < 0 || p->sinks < 0 || p->window > 1 << 30 || p->sinks > 1 << 30) return RINGATTN_ERR_SHAPE;
  if ((p->window > 0 && !p->causal) || (p->sinks > 0 && p->window == 0)) return RINGATTN_ERR_SHAPE;
  if (p->flags & ~(RINGATTN_FLAG_PAGED_PARTIALS | RINGATTN_FLAG_PAGED_KEEP_PRESENT)) return RINGATTN_ERR_SHAPE;
  if (!std::isfinite(p->softmax_scale)) return RINGATTN_ERR_SHAPE;
  return RINGATTN_OK;
}

// The workspace: counters, which are 0 between calls; then the parts of row tiles that several workgroups share.  A call that selects tokens
// to keep has its counts where the parts lie.
constexpr size_t kCounterBytes = rp::kWeightUnits * sizeof(int);
static_assert(rp::kWeightUnits >= 2 * rp::kFewWorkgroups && rp::kWeightUnits * rp::kManyKeys <= rp::kFewSlots * rp::kFewRows * 64);
size_t few_stat_bytes() { return (size_t)rp::kFewSlots * rp::kFewRows * sizeof(float2); }
size_t many_stat_bytes() { return (size_t)rp::kManySlots * rp::kManyRows * sizeof(float2); }
size_t few_o_bytes(int dim) { return (size_t)rp::kFewSlots * rp::kFewRows * dim * sizeof(float); }
size_t many_o_bytes(int dim) { return (size_t)rp::kManySlots * rp::kManyRows * dim * sizeof(float); }
size_t workspace_bytes(int dim) { return kCounterBytes + few_stat_bytes() + many_stat_bytes() + few_o_bytes(dim) + many_o_bytes(dim); }

// The sequences of a call.
int check_cache(const ringattn_paged_plan* pl, const ringattn_paged_cache* c, bool needs_v, bool needs_starts) {
  if (!c) return RINGATTN_ERR_NULL;
  if (!c->k || (needs_v && !c->v) || !c->page_table || !c->kv_lens || (needs_starts && !c->q_starts)) return RINGATTN_ERR_NULL;
  if (c->batch < 0 || c->batch > pl->p.max_batch) return RINGATTN_ERR_SHAPE;
  if (c->pages < 1 || c->table_pages < 1 || (int64_t)c->table_pages * pl->p.page_size > (int64_t)1 << 30) return RINGATTN_ERR_SHAPE;
  if (c->table_stride < c->table_pages || c->table_stride > (int64_t)1 << 40) return RINGATTN_ERR_SHAPE;
  const int64_t most = (int64_t)1 << 40;  // (so that a place in the pool, in bytes, is below 2^62)
  if ((double)c->pages * (double)c->page_stride > (double)((int64_t)1 << 60)) return RINGATTN_ERR_SHAPE;
  if (c->token_stride < pl->p.dim || c->token_stride > 1 << 24 || c->page_stride < pl->p.dim || c->page_stride > most / 2 ||
      c->head_stride < pl->p.dim || c->head_stride > most)
    return RINGATTN_ERR_SHAPE;
  if ((c->token_stride | c->page_stride | c->head_stride) & 7) return RINGATTN_ERR_ALIGN;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->page_table, 4) || !aligned(c->kv_lens, 4) || !aligned(c->q_starts, 4))
    return RINGATTN_ERR_ALIGN;
  return RINGATTN_OK;
}
// Rows of a call's own tensors, by strides in elements of which `unit` make 16 bytes; written ones may not lie on each other.
int check_rows(const ringattn_paged_plan* pl, int tokens, int heads, int64_t ts, int64_t hs, int unit, bool written) {
  if (tokens < 0 || tokens > pl->p.max_tokens) return RINGATTN_ERR_SHAPE;
  const int64_t most = (int64_t)1 << 36;
  if (ts < 0 || hs < 0 || ts > most || hs > most) return RINGATTN_ERR_SHAPE;
  if ((ts | hs) & (unit - 1)) return RINGATTN_ERR_ALIGN;
  const int64_t dim = pl->p.dim, heads_span = heads > 1 ? (heads - 1) * hs + dim : dim;
  const double tokens_span = (double)(tokens - 1) * (double)ts + dim;  // (may pass 64 bits)
  if (written && ((tokens > 1 && ts < dim) || (heads > 1 && hs < dim) || (tokens > 1 && heads > 1 && ts < heads_span && (double)hs < tokens_span)))
    return RINGATTN_ERR_SHAPE;
  return RINGATTN_OK;
}
#define RP_CHECK(expr)                            \
  do {                                            \
    const int rc__ = (expr);                      \
    if (rc__ != RINGATTN_OK) return rc__;         \
  } while (0)
#define RP_HIP(expr)                                                \
  do {                                                              \
    const hipError_t e__ = (expr);                                  \
    if (e__ != hipSuccess) return ringattn::hip_failed(e__);        \
  } while (0)

rp::Cache cache_of(const ringattn_paged_plan* pl, const ringattn_paged_cache* c, int tokens) {
  rp::Cache x;
  std::memset(&x, 0, sizeof(x));
  x.k = (char*)c->k;
  x.v = (char*)c->v;
  x.page_stride = c->page_stride * 2;
  x.head_stride = c->head_stride * 2;
  x.token_stride = (int)(c->token_stride * 2);
  x.pages = c->pages;
  x.table = c->page_table;
  x.table_stride = c->table_stride;
  x.table_pages = c->table_pages;
  x.page_shift = pl->page_shift;
  x.lens = c->kv_lens;
  x.starts = c->q_starts;
  x.batch = c->batch;
  x.tokens = tokens;
  return x;
}

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace

extern "C" {

size_t ringattn_paged_workspace_bytes(const ringattn_paged_params* params) {
  return validate(params) == RINGATTN_OK ? workspace_bytes(params->dim) : 0;
}

int ringattn_paged_plan_create(const ringattn_paged_params* params, void* workspace, size_t workspace_bytes_, ringattn_paged_plan** plan_out) {
  if (!plan_out) return RINGATTN_ERR_NULL;
  *plan_out = nullptr;
  RP_CHECK(validate(params));
  const size_t need = workspace_bytes(params->dim);
  if (workspace) {
    if (workspace_bytes_ < need) return RINGATTN_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return RINGATTN_ERR_ALIGN;
  }
  ringattn_paged_plan* pl = new (std::nothrow) ringattn_paged_plan();
  if (!pl) return RINGATTN_ERR_ALLOC;
  pl->p = *params;
  pl->kv_heads = params->kv_heads > 0 ? params->kv_heads : params->heads;
  pl->scale = params->softmax_scale > 0.f ? params->softmax_scale : 1.0f / std::sqrt((float)params->dim);
  pl->page_shift = __builtin_ctz((unsigned)params->page_size);
  pl->ws = workspace;
  if (!workspace) {
    hipError_t e = hipMalloc(&pl->ws, need);
    if (e == hipSuccess) {
      hipStream_t own = nullptr;  // (a stream of its own: nothing else is waited for)
      e = hipStreamCreateWithFlags(&own, hipStreamNonBlocking);
      if (e == hipSuccess) {
        e = hipMemsetAsync(pl->ws, 0, kCounterBytes, own);
        if (e == hipSuccess) e = hipStreamSynchronize(own);
        (void)hipStreamDestroy(own);
      }
      if (e != hipSuccess) (void)hipFree(pl->ws);
    }
    if (e != hipSuccess) {
      delete pl;
      const int rc = ringattn::hip_failed(e);
      return e == hipErrorOutOfMemory ? RINGATTN_ERR_ALLOC : rc;
    }
    pl->own_ws = true;
  }
  try {
    std::lock_guard<std::mutex> lk(g_paged_mu);
    g_paged_plans.insert(pl);
  } catch (...) {
    if (pl->own_ws) (void)hipFree(pl->ws);
    delete pl;
    return RINGATTN_ERR_ALLOC;
  }
  *plan_out = pl;
  return RINGATTN_OK;
}

int ringattn_paged_plan_destroy(ringattn_paged_plan* plan) {
  {
    std::lock_guard<std::mutex> lk(g_paged_mu);
    if (!plan || g_paged_plans.erase(plan) == 0) return RINGATTN_ERR_PLAN;
  }
  int rc = RINGATTN_OK;
  if (plan->own_ws) {
    const hipError_t e = hipFree(plan->ws);
    if (e != hipSuccess) rc = ringattn::hip_failed(e);
  }
  delete plan;
  return rc;
}

int ringattn_paged_append(ringattn_paged_plan* plan, const ringattn_paged_cache* cache, const void* k_new, const void* v_new, int tokens,
                          int64_t token_stride, int64_t head_stride, float* scores, void* stream) {
  if (!plan_ok(plan)) return RINGATTN_ERR_PLAN;
  RP_CHECK(check_cache(plan, cache, true, true));
  if (!k_new || !v_new) return RINGATTN_ERR_NULL;
  RP_CHECK(check_rows(plan, tokens, plan->kv_heads, token_stride, head_stride, 8, false));
  if (!aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(scores, 4)) return RINGATTN_ERR_ALIGN;
  rp::AppendArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = cache_of(plan, cache, tokens);
  a.k = (const char*)k_new;
  a.v = (const char*)v_new;
  a.ts = token_stride * 2;
  a.hs = head_stride * 2;
  a.scores = scores;
  a.kv_heads = plan->kv_heads;
  RP_HIP(rp::launch_paged_append(a, plan->p.dim, (hipStream_t)stream));
  return RINGATTN_OK;
}

int ringattn_paged_fwd(ringattn_paged_plan* plan, const ringattn_paged_cache* cache, const void* q, int tokens, int64_t q_token_stride,
                       int64_t q_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, void* stream_) {
  if (!plan_ok(plan)) return RINGATTN_ERR_PLAN;
  RP_CHECK(check_cache(plan, cache, true, true));
  if (!q || !out || !lse) return RINGATTN_ERR_NULL;
  const bool fp32 = (plan->p.flags & RINGATTN_FLAG_PAGED_PARTIALS) != 0;
  RP_CHECK(check_rows(plan, tokens, plan->p.heads, q_token_stride, q_head_stride, 8, false));
  RP_CHECK(check_rows(plan, tokens, plan->p.heads, out_token_stride, out_head_stride, fp32 ? 4 : 8, true));
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(lse, 4)) return RINGATTN_ERR_ALIGN;
  if (tokens == 0 || cache->batch == 0) return RINGATTN_OK;
  hipStream_t stream = (hipStream_t)stream_;
  const int kv = plan->kv_heads, group = plan->p.heads / kv;
  rp::AttendArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = cache_of(plan, cache, tokens);
  a.q = (const char*)q;
  a.out = (char*)out;
  a.lse = lse;
  char* ws = (char*)plan->ws;
  a.few.arrived = (int*)ws;
  a.few.stat = (float2*)(ws += kCounterBytes);
  a.many.stat = (float2*)(ws += few_stat_bytes());
  a.few.o = (float*)(ws += many_stat_bytes());
  a.many.o = (float*)(ws += few_o_bytes(plan->p.dim));
  a.q_ts = q_token_stride * 2;
  a.q_hs = q_head_stride * 2;
  a.o_ts = out_token_stride * (fp32 ? 4 : 2);
  a.o_hs = out_head_stride * (fp32 ? 4 : 2);
  a.kv_heads = kv;
  a.group = group;
  a.by_group = ringattn::divisor(group);
  a.by_kv_heads = ringattn::divisor(kv);
  a.scale_log2 = plan->scale * kLog2e;
  a.causal = plan->p.causal != 0;
  a.window = plan->p.window;
  a.sinks = plan->p.sinks;
  a.out_fp32 = fp32;
  const int64_t rows = (int64_t)tokens * group, sequences = cache->batch < tokens ? cache->batch : tokens;
  // What sequences see at most, in key tiles, and their row tiles if all have few rows; in units so large that 2^30 suffice for both.
  const int64_t few_tiles = rows / rp::kFewRows + sequences;
  const int64_t see = ((int64_t)cache->table_pages * plan->p.page_size + rp::kKeyTile - 1) / rp::kKeyTile + rp::kFewSmall;
  const int64_t in_window = a.window > 0 ? (a.window + rp::kManyRows + (int64_t)a.sinks) / rp::kKeyTile + 3 : see, most = see < in_window ? see : in_window;
  // More rows are few where that cannot make more work than kFewMore key tiles a workgroup, whose parts are fewer and smaller.
  const bool little = few_tiles * kv * most <= (int64_t)rp::kFewMore * rp::kFewWorkgroups;
  a.few_most = few_most(tokens, cache->batch, little ? rp::kFewRowsMore : cache->batch == 1 ? rp::kFewRowsAlone : rp::kFewRowsMost);
  while (few_tiles * kv * (((see - 1) >> a.few_shift) + 1) > (int64_t)1 << 30) ++a.few_shift;
  // Row tiles of any lengths: every sequence of many rows begins one, and 256 rows more another.  Where they alone fill the compute units
  // their keys are not shared out, unless some sequence may be much longer than others; else there is a share each, and no more besides than
  // are due.  (Us with and without shares, 32 heads on 8 of 128: a chunk of 512 over 8 K, 64 row tiles, 91 and 193; 509 tokens over 2.3 K,
  // 16 heads on 4, 34 and 65; prompts of 1 K, 32 heads, 128 row tiles, 50 and 44; eight chunks of 512, one over 32 K, seven over 1 K, 512
  // row tiles, 347 and 742; 16 of them, one over 16 K, 1024 row tiles, 410 and 397.)
  const int64_t might = rows / ((int64_t)a.few_most + 1), with_many = might < sequences ? might : sequences;
  const int64_t tiles = with_many > 0 ? rows / rp::kManyRows + with_many : 0, due = rp::kManyWorkgroups / kv + 1;
  a.many_cut = tiles > 0 && rows / rp::kManyRows * kv < (most >= 512 ? 4 * rp::kManyWorkgroups : rp::kManyWorkgroups);
  const int64_t places = tiles + (a.many_cut ? due : 0);
  // Workgroups of few rows first; of a sequence alone, whose rows are many if q is full, last, where they cost a full one next to nothing (us
  // with and without them: 4096 tokens over 32 K, 32 heads 1867 and 1867; with a window of 1024, 8 KV heads 94.9 and 94.2).
  a.few_begin = sequences == 1 ? (int)(places * kv) : 0;
  RP_HIP(rp::launch_paged_attend(a, plan->p.dtype, plan->p.dim, places, tiles < due ? tiles : due, stream));
  return RINGATTN_OK;
}

int ringattn_paged_weights(ringattn_paged_plan* plan, const ringattn_paged_cache* cache, const void* q, int tokens, int64_t q_token_stride,
                           int64_t q_head_stride, const float* lse, float* scores, void* stream) {
  if (!plan_ok(plan)) return RINGATTN_ERR_PLAN;
  RP_CHECK(check_cache(plan, cache, false, true));
  if (!q || !lse || !scores) return RINGATTN_ERR_NULL;
  RP_CHECK(check_rows(plan, tokens, plan->p.heads, q_token_stride, q_head_stride, 8, false));
  if (!aligned(q, 16) || !aligned(lse, 4) || !aligned(scores, 4)) return RINGATTN_ERR_ALIGN;
  if (tokens == 0 || cache->batch == 0) return RINGATTN_OK;
  rp::WeightsArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = cache_of(plan, cache, tokens);
  a.q = (const char*)q;
  a.lse = lse;
  a.scores = scores;
  a.q_ts = q_token_stride * 2;
  a.q_hs = q_head_stride * 2;
  a.kv_heads = plan->kv_heads;
  a.group = plan->p.heads / plan->kv_heads;
  a.by_group = ringattn::divisor(a.group);
  a.scale_log2 = plan->scale * kLog2e;
  a.causal = plan->p.causal != 0;
  a.window = plan->p.window;
  a.sinks = plan->p.sinks;
  // One sequence has one launch: of few rows if q has few; else of many, also where its new tokens turn out to be fewer than the rows of q, so
  // that none count as few.  (Us over 32 K, 32 heads on 8, new tokens in q of as many rows and of 512: 1 22 and 68, 16 33 and 67, 48 68 and 75.
  // A second launch in every call of one sequence would take some 4.)
  a.few_most = cache->batch == 1 && (int64_t)tokens * a.group > rp::kWeightFewRowsMost ? 0 : few_most(tokens, cache->batch, rp::kWeightFewRowsMost);
  a.arrived = (int*)plan->ws;
  a.parts = (float*)((char*)plan->ws + kCounterBytes);
  a.q_even = 32 % a.group == 0 && a.q_ts < 1 << 25 && a.q_hs < 1 << 25 && (int64_t)a.group * tokens < 1 << 29;
  RP_HIP(rp::launch_paged_weights(a, plan->p.dtype, plan->p.dim, (hipStream_t)stream));
  return RINGATTN_OK;
}

int ringattn_paged_evict(ringattn_paged_plan* plan, const ringattn_paged_cache* cache, float* scores, const int* kept_table, int kept_pages,
                         int64_t kept_stride, int budget, int keep_first, int keep_last, int* kept, int* kept_lens, void* stream) {
  if (!plan_ok(plan)) return RINGATTN_ERR_PLAN;
  RP_CHECK(check_cache(plan, cache, true, false));
  if (!scores || !kept_table || !kept || !kept_lens) return RINGATTN_ERR_NULL;
  if (budget < 1 || keep_first < 0 || keep_last < 0 || (int64_t)keep_first + keep_last > budget) return RINGATTN_ERR_SEQLEN;
  if (kept_pages < 1 || kept_stride < kept_pages || kept_stride > (int64_t)1 << 40) return RINGATTN_ERR_SHAPE;
  if ((int64_t)kept_pages * plan->p.page_size < budget || (int64_t)kept_pages * plan->p.page_size > (int64_t)1 << 30) return RINGATTN_ERR_SHAPE;
  if (!aligned(scores, 4) || !aligned(kept_table, 4) || !aligned(kept, 4) || !aligned(kept_lens, 4)) return RINGATTN_ERR_ALIGN;
  if (cache->batch == 0) return RINGATTN_OK;
  rp::EvictArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = cache_of(plan, cache, 0);
  a.scores = scores;
  a.kept_table = kept_table;
  a.kept_stride = kept_stride;
  a.kept_pages = kept_pages;
  a.budget = budget;
  a.first = keep_first;
  a.last = keep_last;
  a.present = (plan->p.flags & RINGATTN_FLAG_PAGED_KEEP_PRESENT) != 0;
  a.kept = kept;
  a.kept_lens = kept_lens;
  a.workspace = (char*)plan->ws + kCounterBytes;
  a.workspace_bytes = workspace_bytes(plan->p.dim) - kCounterBytes;
  a.kv_heads = plan->kv_heads;
  RP_HIP(rp::launch_paged_evict(a, plan->p.dim, (hipStream_t)stream));
  return RINGATTN_OK;
}

}  // extern "C"
