// Rotary positions: launch arguments, and a thread's part of a row.
//
// Pair i of a row's first `turned` columns turns by pos * f_i.  The angle is taken as a part of a full turn: f_i comes as 2^64 f_i / 2 pi, an
// integer, and pos * f_i mod 2^64 is the part of a turn, exactly, for any position of 32 bits; its upper half, as a number in [-1/2, 1/2), is off
// by 2^-26 (32 bits of fp32 in its place are off by pos * f_i * 2^-24: 0.06 of a radian at a million tokens).
#pragma once
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
