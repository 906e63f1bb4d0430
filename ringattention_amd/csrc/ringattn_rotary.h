// Rotary positions: launch arguments, and a thread's part of a row.
//
// Pair i of a row's first `turned` columns turns by pos * f_i.  The angle is taken as a part of a full turn: f_i comes as 2^64 f_i / 2 pi, an
// integer, and pos * f_i mod 2^64 is the part of a turn, exactly, for any position of 32 bits; its upper half, as a number in [-1/2, 1/2), is off
// by 2^-26 (32 bits of fp32 in its place are off by pos * f_i * 2^-24: 0.06 of a radian at a million tokens).
#pragma once
#include <cstdlib>

#include "ringattn.h"
#include "ringattn_paged.h"

namespace ringattn {
namespace rotary {

struct Turns {
  const uint64_t* turns;  // [turned / 2]
  float factor;           // of the turned columns
  int turned;             // columns, the first ones; a multiple of 16
  int back;               // by minus the angles
};

// What is wrong with a caller's rotary, or what the kernels are told of it.
int check(const ringattn_rotary* r, int dim, Turns* out);

// Rows [tokens, heads, dim] of 16-bit values: the first one, and elements between tokens and heads.
struct RowsAt {
  const void* at;
  int64_t ts, hs;
  int heads;
};
// Whether a row of the one tensor, none of whose own lie on each other, lies on a row of the other, as far as that can be told: they lie apart; or a
// token's rows do, modulo the distance of tokens, which is the same for both (a fused projection's Q, K and V); or both distances are the same and two
// rows come within dim of each other, or none do.
enum class Meet { kApart, kMeet, kUnknown };
inline Meet rows_meet(const RowsAt& a, const RowsAt& b, int tokens, int dim) {
  const double fa = (double)(uintptr_t)a.at, fb = (double)(uintptr_t)b.at;
  auto bytes = [&](const RowsAt& x) { return 2. * ((double)(tokens - 1) * (double)x.ts + (double)(x.heads - 1) * (double)x.hs + dim); };
  if (fa + bytes(a) <= fb || fb + bytes(b) <= fa) return Meet::kApart;
  const int64_t d = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at) / 2;  // elements from a's first row to b's
  if (d > -dim && d < dim) return Meet::kMeet;                         // (the first rows themselves)
  const int64_t none = INT64_MAX / 4;                                  // the distance of what there is one of
  if (tokens > 1 && (a.ts != b.ts || a.ts == 0)) return Meet::kUnknown;
  const int64_t ts = tokens > 1 ? a.ts : none, hs = a.heads > 1 ? a.hs : b.heads > 1 ? b.hs : none;
  auto block = [&](const RowsAt& x) { return x.heads > 1 ? (x.heads - 1) * x.hs + dim : dim; };  // of a token
  const int64_t from = (d % ts + ts) % ts;                                                        // where b's begins in a's distance of tokens
  if (from >= block(a) && from + block(b) <= ts) return Meet::kApart;
  if ((a.heads > 1 && b.heads > 1 && a.hs != b.hs) || hs == 0) return Meet::kUnknown;
  // the rows that come nearest: so many tokens and heads of a's further on, the larger distance first
  const bool by_token = ts > hs;
  const int64_t large = by_token ? ts : hs, small = by_token ? hs : ts;
  auto in_range = [&](int64_t n, bool of_tokens) { return of_tokens ? n > -tokens && n < tokens : n > -b.heads && n < a.heads; };
  for (int64_t i = d / large - 2; i <= d / large + 2; ++i) {
    if (!in_range(i, by_token)) continue;
    const int64_t left = d - i * large;
    for (int64_t j = left / small - 1; j <= left / small + 1; ++j)
      if (in_range(j, !by_token) && std::llabs(left - j * small) < dim) return Meet::kMeet;
  }
  return a.heads >= b.heads ? Meet::kApart : Meet::kUnknown;  // (b's heads may reach past a's distance of tokens)
}

struct Rows {
  const char* in;
  char* out;
  int64_t in_bs, in_hs, in_ts, out_bs, out_hs, out_ts;  // bytes
};
struct ApplyArgs {
  Turns r;
  Rows x[2];
  int heads0, heads;       // of the first tensor, of both
  int tokens;
  const int* positions;    // NULL: a row's number
  int64_t position_stride; // between batches
};
hipError_t launch_apply(const ApplyArgs& a, int dtype, int dim, bool interleaved, int batch, hipStream_t stream);

struct AppendArgs {
  paged::Cache c;
  Turns r;
  const char *q, *k, *v;
  char* q_out;
  int64_t q_ts, q_hs, o_ts, o_hs, ts, hs;  // bytes: of q, of q_out, of k and v
  const int* positions;                    // [tokens]; NULL: a token's place in its sequence
  float* scores;                           // [pages, kv_heads, page] or NULL
  int heads, kv_heads;
  int rows_each;                           // rows (q, k and v heads of a token) of a wave
};
hipError_t launch_append(const AppendArgs& a, int dtype, int dim, bool interleaved, hipStream_t stream);

// Sixteen columns of a row, as two pieces of eight: a thread's eight pairs, or sixteen columns that stay.  Pairs are columns i and
// i + turned / 2, so that the pieces lie half the turned part apart, or 2 i and 2 i + 1.
struct Part {
  int at0, at1;  // bytes from the row's first column
  bool turns;
};
template <bool INTERLEAVED> static __device__ __forceinline__ Part part_of(const Turns& r, int piece) {
  Part p;
  p.turns = piece * 16 < r.turned;
  const bool halves = p.turns && !INTERLEAVED;
  p.at0 = halves ? 16 * piece : 32 * piece;
  p.at1 = halves ? 16 * piece + r.turned : 32 * piece + 16;
  return p;
}
struct Angles {
  float c[8], s[8];
};
static __device__ __forceinline__ void angles_of(Angles& x, const Turns& r, int piece, int64_t pos) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t turn = (uint64_t)pos * r.turns[8 * piece + i];
    float t = (float)(int)(turn >> 32) * 0x1p-32f;
    t = r.back ? -t : t;
    x.c[i] = __builtin_amdgcn_cosf(t) * r.factor;  // (of turns)
    x.s[i] = __builtin_amdgcn_sinf(t) * r.factor;
  }
}
template <int DT, bool INTERLEAVED>
static __device__ __forceinline__ void turn(s16x8& x0, s16x8& x1, const Angles& g) {
  using vec8 = typename Elem<DT>::vec8;
  using T = typename Elem<DT>::type;
  vec8 a = __builtin_bit_cast(vec8, x0), b = __builtin_bit_cast(vec8, x1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (INTERLEAVED) {
      vec8& v = i < 4 ? a : b;
      const float p = (float)v[2 * (i & 3)], q = (float)v[2 * (i & 3) + 1];
      v[2 * (i & 3)] = (T)__builtin_fmaf(p, g.c[i], -(q * g.s[i]));
      v[2 * (i & 3) + 1] = (T)__builtin_fmaf(q, g.c[i], p * g.s[i]);
    } else {
      const float p = (float)a[i], q = (float)b[i];
      a[i] = (T)__builtin_fmaf(p, g.c[i], -(q * g.s[i]));
      b[i] = (T)__builtin_fmaf(q, g.c[i], p * g.s[i]);
    }
  }
  x0 = __builtin_bit_cast(s16x8, a);
  x1 = __builtin_bit_cast(s16x8, b);
}

}  // namespace rotary
}  // namespace ringattn
