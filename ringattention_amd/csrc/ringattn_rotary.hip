// gfx950 (CDNA4) kernels: rotary positions, of a ring's tensors (ringattn_rotary_apply) and of new tokens on their way into a paged cache
// (ringattn_paged_append_rotary).  Copies with some arithmetic: memory bounds them where there are many rows, a launch where few.
//
//   rotary_kernel        : a thread has sixteen columns of a row, eight pairs; their angles cost it less than the memory takes (32 K tokens, 32/8
//       heads x 128: 111 us, 6.0 TB/s read and written; two, four, eight heads a thread with their angles in common 117, 122, 127).
//   rotary_append_kernel : a wave has a token, D / 16 lanes a row: Q's heads to their output, K's turned and V's as they are to the page.  8 K tokens of
//       prompts, 32 heads each 81 us, 5.0 TB/s; one token a sequence a launch and three loads one behind the other.
#include "ringattn_rotary.h"

#include <cmath>
#include <cstring>
#include <utility>

namespace ringattn {
namespace rotary {

template <int DT, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const ApplyArgs a) {
  constexpr int PIECES = D / 16;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int piece = (int)(item % PIECES);
  const int64_t t = item / PIECES;
  if (t >= a.tokens) return;
  const int b = blockIdx.z, h = blockIdx.y;
  const Part p = part_of<INTERLEAVED>(a.r, piece);
  const bool second = h >= a.heads0;
  const Rows& x = a.x[second ? 1 : 0];
  const int head = second ? h - a.heads0 : h;
  const char* from = x.in + b * x.in_bs + head * x.in_hs + t * x.in_ts;
  char* to = x.out + b * x.out_bs + head * x.out_hs + t * x.out_ts;
  if (!p.turns && from == to) return;
  s16x8 x0 = *(const s16x8*)(from + p.at0), x1 = *(const s16x8*)(from + p.at1);
  if (p.turns) {
    Angles g;
    angles_of(g, a.r, piece, a.positions ? (int64_t)a.positions[b * a.position_stride + t] : t);
    turn<DT, INTERLEAVED>(x0, x1, g);
  }
  *(s16x8*)(to + p.at0) = x0;
  *(s16x8*)(to + p.at1) = x1;
}

template <int DT, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_append_kernel(const AppendArgs a) {
  constexpr int PIECES = D / 16, AT_ONCE = 64 / PIECES;
  const int lane = threadIdx.x & 63;
  const int t = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
  if (t >= a.c.tokens) return;
  // the sequence that token t is of: the last one that begins at or before it; its lengths and starts are held to the same as everywhere.  Up to 64
  // of them, then up to 64 sequences, at a look, a lane each: two loads one behind the other, not twelve.
  const int step = (a.c.batch + 63) / 64;
  auto last_of = [&](int first, int by, int count) {
    const int i = first + lane * by;
    const uint64_t begun = __builtin_amdgcn_ballot_w64(lane < count && i < a.c.batch && a.c.starts[min(i, a.c.batch)] <= t);
    return begun == 0 ? first : first + by * (63 - __builtin_clzll(begun));
  };
  int lo = last_of(0, step, 64);
  if (step > 1) lo = last_of(lo, 1, step);
  lo = __builtin_amdgcn_readfirstlane(lo);
  const paged::Seq s = paged::uniform(paged::seq_of(a.c, lo));
  const int i = t - s.start, key = s.len - s.n + i;
  if (i < 0 || i >= s.n) return;  // in front of the first, behind the last
  int page = key >= 0 ? a.c.table[lo * a.c.table_stride + (key >> a.c.page_shift)] : -1;  // (more new tokens than there are tokens)
  page = __builtin_amdgcn_readfirstlane(page);
  const bool there = (unsigned)page < (unsigned)a.c.pages;
  const int piece = lane % PIECES;
  const Part p = part_of<INTERLEAVED>(a.r, piece);
  Angles g;
  if (p.turns) angles_of(g, a.r, piece, a.positions ? a.positions[t] : key);
  const int row_begin = blockIdx.y * a.rows_each, rows = min(row_begin + a.rows_each, a.heads + 2 * a.kv_heads);
  for (int row = row_begin + lane / PIECES; row < rows; row += AT_ONCE) {
    const bool of_q = row < a.heads, of_v = row >= a.heads + a.kv_heads;
    const int head = of_q ? row : of_v ? row - a.heads - a.kv_heads : row - a.heads;
    if (!of_q && !there) continue;
    const char* from = of_q ? a.q + t * a.q_ts + head * a.q_hs : (of_v ? a.v : a.k) + t * a.ts + head * a.hs;
    char* to = of_q ? a.q_out + t * a.o_ts + head * a.o_hs : (of_v ? a.c.v : a.c.k) + paged::page_row(a.c, page, head, key);
    s16x8 x0 = *(const s16x8*)(from + p.at0), x1 = *(const s16x8*)(from + p.at1);
    if (p.turns && !of_v) turn<DT, INTERLEAVED>(x0, x1, g);
    *(s16x8*)(to + p.at0) = x0;
    *(s16x8*)(to + p.at1) = x1;
    if (of_v && piece == 0 && a.scores) a.scores[(((int64_t)page * a.kv_heads + head) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1))] = 0.f;
  }
}

#define RA_ROTARY_FORMS(LAUNCH)                                             \
  do {                                                                      \
    if (dtype == 0 && dim == 64 && !interleaved) LAUNCH(0, 64, false);      \
    else if (dtype == 0 && dim == 64) LAUNCH(0, 64, true);                  \
    else if (dtype == 1 && dim == 64 && !interleaved) LAUNCH(1, 64, false); \
    else if (dtype == 1 && dim == 64) LAUNCH(1, 64, true);                  \
    else if (dtype == 0 && dim == 128 && !interleaved) LAUNCH(0, 128, false); \
    else if (dtype == 0 && dim == 128) LAUNCH(0, 128, true);                \
    else if (dtype == 1 && dim == 128 && !interleaved) LAUNCH(1, 128, false); \
    else if (dtype == 1 && dim == 128) LAUNCH(1, 128, true);                \
    else return hipErrorInvalidValue;                                       \
  } while (0)

hipError_t launch_apply(const ApplyArgs& a, int dtype, int dim, bool interleaved, int batch, hipStream_t stream) {
  const int64_t blocks = ((int64_t)a.tokens * (dim / 16) + 255) / 256;
  if (blocks <= 0 || batch <= 0) return hipSuccess;
  if (blocks > INT32_MAX || a.heads > 65535 || batch > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)a.heads, (unsigned)batch);
#define RA_LAUNCH(DT_, D_, I_) rotary_kernel<DT_, D_, I_><<<grid, 256, 0, stream>>>(a)
  RA_ROTARY_FORMS(RA_LAUNCH);
#undef RA_LAUNCH
  return hipGetLastError();
}

hipError_t launch_append(const AppendArgs& args, int dtype, int dim, bool interleaved, hipStream_t stream) {
  AppendArgs a = args;
  if (a.c.tokens <= 0 || a.c.batch <= 0) return hipSuccess;
  const int rows = a.heads + 2 * a.kv_heads;
  // A wave has all rows of its token where there are many tokens; of few, so many that there are some 2048 waves.  (Us so and with all, 32 heads on 8: one
  // token 2.8 and 4.4, 48 3.0 and 4.8, 200 3.6 and 5.1, 500 4.4 and 5.4; 3000 are the same.)
  const int at_once = 1024 / dim, rounds = (rows + at_once - 1) / at_once, wanted = 2048 / a.c.tokens;
  const int waves = wanted < 1 ? 1 : wanted < rounds ? wanted : rounds;
  a.rows_each = (rounds + waves - 1) / waves * at_once;
  const dim3 grid((unsigned)((a.c.tokens + 3) / 4), (unsigned)((rows + a.rows_each - 1) / a.rows_each));
#define RA_LAUNCH(DT_, D_, I_) rotary_append_kernel<DT_, D_, I_><<<grid, 256, 0, stream>>>(a)
  RA_ROTARY_FORMS(RA_LAUNCH);
#undef RA_LAUNCH
  return hipGetLastError();
}

int check(const ringattn_rotary* r, int dim, Turns* out) {
  if (!r || !r->turns) return RINGATTN_ERR_NULL;
  if (r->rotary_dim < 16 || r->rotary_dim > dim || r->rotary_dim % 16 != 0) return RINGATTN_ERR_DIM;
  if (!std::isfinite(r->factor) || r->factor < 0.f) return RINGATTN_ERR_SHAPE;
  if ((uintptr_t)r->turns & 7) return RINGATTN_ERR_ALIGN;
  *out = Turns{r->turns, r->factor > 0.f ? r->factor : 1.f, r->rotary_dim, r->inverse != 0};
  return RINGATTN_OK;
}

namespace {

// A tensor's rows: strides of dimensions that have one entry count for nothing.
struct Extent {
  int64_t n[3], stride[3];  // elements; batch, head, token
  int dim;
  bool in_range() const {
    for (int i = 0; i < 3; ++i)
      if (n[i] > 1 && (stride[i] < 0 || stride[i] > (int64_t)1 << 36)) return false;
    return true;
  }
  bool in_pieces() const {
    for (int i = 0; i < 3; ++i)
      if (n[i] > 1 && (stride[i] & 7)) return false;
    return true;
  }
  double span() const {  // elements from the first to behind the last (may pass 64 bits)
    double x = dim;
    for (int i = 0; i < 3; ++i) x += (double)(n[i] - 1) * (double)(n[i] > 1 ? stride[i] : 0);
    return x;
  }
  // No row on another: each dimension steps over what lies within the smaller ones.
  bool apart() const {
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
      for (int j = i + 1; j < 3; ++j)
        if ((n[order[j]] > 1 ? stride[order[j]] : -1) < (n[order[i]] > 1 ? stride[order[i]] : -1)) std::swap(order[i], order[j]);
    double within = dim;
    for (int i = 0; i < 3; ++i) {
      const int d = order[i];
      if (n[d] < 2) continue;
      if ((double)stride[d] < within) return false;
      within += (double)(n[d] - 1) * (double)stride[d];
    }
    return true;
  }
};

// Whether the output of one tensor of a call can be shown to lie on rows of the other one, by what lies in each batch (rows_meet).
struct Tensor {
  const void* at;
  int64_t bs, hs, ts;
  int heads;
};
bool lies_on(const Tensor& out, const Tensor& other, int batch, int tokens, int dim) {
  if (batch > 1 && (out.bs != other.bs || out.bs == 0)) return false;
  const RowsAt rows{out.at, out.ts, out.hs, out.heads};
  const int64_t d = (int64_t)((uintptr_t)other.at - (uintptr_t)out.at) / 2, near = batch > 1 ? d / out.bs : 0;
  for (int64_t i = near - 2; i <= near + 2; ++i) {
    if (i <= -batch || i >= batch) continue;
    const uintptr_t at = (uintptr_t)other.at - (uintptr_t)(batch > 1 ? i * out.bs * 2 : 0);  // as it lies to the output i batches on
    if (rows_meet(rows, RowsAt{(const void*)at, other.ts, other.hs, other.heads}, tokens, dim) == Meet::kMeet) return true;
  }
  return false;
}

}  // namespace

}  // namespace rotary
}  // namespace ringattn

extern "C" {

int ringattn_rotary_turns(const double* radians, int n, uint64_t* turns) {
  if (!radians || !turns) return RINGATTN_ERR_NULL;
  if (n < 0) return RINGATTN_ERR_SHAPE;
  for (int i = 0; i < n; ++i)
    if (!std::isfinite(radians[i])) return RINGATTN_ERR_SHAPE;
  for (int i = 0; i < n; ++i) {
    long double t = (long double)radians[i] / 6.283185307179586476925286766559L;
    t -= floorl(t);  // whole turns are none
    const long double x = roundl(t * 18446744073709551616.0L);
    turns[i] = x >= 18446744073709551616.0L ? 0 : (uint64_t)x;
  }
  return RINGATTN_OK;
}

int ringattn_rotary_apply(const ringattn_rotary* rotary, int dim, int dtype, const ringattn_rows* tensors, int count, int batch, int tokens,
                          const int* positions, int64_t position_stride, void* stream) {
  namespace rr = ringattn::rotary;
  if (dim != 64 && dim != 128) return RINGATTN_ERR_DIM;
  if (dtype != RINGATTN_DTYPE_FP16 && dtype != RINGATTN_DTYPE_BF16) return RINGATTN_ERR_DTYPE;
  rr::ApplyArgs a;
  std::memset(&a, 0, sizeof(a));
  if (const int rc = rr::check(rotary, dim, &a.r)) return rc;
  if (!tensors) return RINGATTN_ERR_NULL;
  if (count < 1 || count > 2 || batch < 0 || batch > 65535 || tokens < 0 || tokens > 1 << 30) return RINGATTN_ERR_SHAPE;
  if (positions && (position_stride < 0 || position_stride > (int64_t)1 << 40)) return RINGATTN_ERR_SHAPE;
  if ((uintptr_t)positions & 3) return RINGATTN_ERR_ALIGN;
  for (int i = 0; i < count; ++i) {
    const ringattn_rows& x = tensors[i];
    if (x.heads < 1 || x.heads > 65535) return RINGATTN_ERR_SHAPE;
    if (!x.in || !x.out) return RINGATTN_ERR_NULL;
    const rr::Extent in{{batch, x.heads, tokens}, {x.in_batch_stride, x.in_head_stride, x.in_token_stride}, dim};
    const rr::Extent out{{batch, x.heads, tokens}, {x.out_batch_stride, x.out_head_stride, x.out_token_stride}, dim};
    if (!in.in_range() || !out.in_range()) return RINGATTN_ERR_SHAPE;
    if (!in.in_pieces() || !out.in_pieces() || (((uintptr_t)x.in | (uintptr_t)x.out) & 15)) return RINGATTN_ERR_ALIGN;
    if (!out.apart()) return RINGATTN_ERR_SHAPE;
    // the tensor itself, or one that lies elsewhere
    bool same = x.in == x.out;
    for (int d = 0; d < 3; ++d) same = same && (in.n[d] < 2 || in.stride[d] == out.stride[d]);
    const double from = (double)(uintptr_t)x.in, to = (double)(uintptr_t)x.out;
    if (!same && batch > 0 && tokens > 0 && from < to + 2 * out.span() && to < from + 2 * in.span()) return RINGATTN_ERR_SHAPE;
    rr::Rows& r = a.x[i];
    auto bytes = [](const rr::Extent& e, int d) { return e.n[d] > 1 ? e.stride[d] * 2 : 0; };
    r = rr::Rows{(const char*)x.in, (char*)x.out, bytes(in, 0), bytes(in, 1), bytes(in, 2), bytes(out, 0), bytes(out, 1), bytes(out, 2)};
    a.heads += x.heads;
    if (a.heads > 65535) return RINGATTN_ERR_SHAPE;
  }
  // Of two, neither's output has the other's rows: what is in the same place, and what equal strides show, is refused; of other strides it is the caller's to see.
  if (count == 2 && batch > 0 && tokens > 0) {
    if (tensors[0].out == tensors[1].out || tensors[0].out == tensors[1].in || tensors[1].out == tensors[0].in) return RINGATTN_ERR_SHAPE;
    auto in = [](const ringattn_rows& x) { return rr::Tensor{x.in, x.in_batch_stride, x.in_head_stride, x.in_token_stride, x.heads}; };
    auto out = [](const ringattn_rows& x) { return rr::Tensor{x.out, x.out_batch_stride, x.out_head_stride, x.out_token_stride, x.heads}; };
    if (rr::lies_on(out(tensors[0]), out(tensors[1]), batch, tokens, dim) || rr::lies_on(out(tensors[0]), in(tensors[1]), batch, tokens, dim) ||
        rr::lies_on(out(tensors[1]), in(tensors[0]), batch, tokens, dim))
      return RINGATTN_ERR_SHAPE;
  }
  a.heads0 = tensors[0].heads;
  a.tokens = tokens;
  a.positions = positions;
  a.position_stride = position_stride;
  const hipError_t e = rr::launch_apply(a, dtype, dim, rotary->interleaved != 0, batch, (hipStream_t)stream);
  return e == hipSuccess ? RINGATTN_OK : ringattn::hip_failed(e);
}

}  // extern "C"
