// it_rotary.hpp -- rotary positions: the handle, and what the kernels that
// rotate share (the append, the plain rotation, the move of cached rows).
#pragma once
#include <hip/hip_runtime.h>

#include "it_device.hpp"
#include "it_internal.hpp"
#include "it_kv.h"
#include "it_rows.hpp"

struct it_rotary {
  double* turns;   // device [n_dims / 2]: turns per position of each pair, f_p / (2 pi)
  float magnitude; // multiplies cos and sin
  int32_t device;
  int32_t n_dims;
  int32_t layout;  // IT_ROTARY_INTERLEAVED or IT_ROTARY_HALF
};

namespace itkv {

// (cos, sin) of 2 pi turns pos, each within about one fp32 ulp of 1.  The product
// is taken in fp64 (turns' own rounding is all that is lost: 2^-53 of the angle,
// 2^-33 radians at a million positions of the fastest pair) and reduced there exactly: r to the nearest whole turn, then
// to the nearest quarter; the rest, |x| <= pi/4, is rounded to fp32 once, and the
// Taylor sums end where the next term is below 2^-25 at pi/4 (x^11 / 11!, x^12 /
// 12!).  No table: a table of every position would cost a second dependent load
// (and 512 bytes a position at head_dim 128) where this is ~40 instructions per
// pair and token, hidden behind the rows' loads.
__device__ __forceinline__ float2 rotary_angle(double turns, int pos) {
  const double r = fma(turns, double(pos), -__builtin_rint(turns * double(pos)));
  const double quarter = __builtin_rint(4.0 * r);  // -2 .. 2
  const float x = float(fma(-0.25, quarter, r) * 6.283185307179586);
  const float y = x * x;
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f), -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
  const float p = fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f);
  const float s = fmaf(x * y, p, x);
  const int q = int(quarter) & 3;
  const float a = (q & 1) ? s : c, b = (q & 1) ? c : s;
  return make_float2((q == 1 || q == 2) ? -a : a, (q & 2) ? -b : b);
}

// The two elements of a pair turned, each with the same two roundings in every
// kernel: a row's result does not depend on which of them took it.
__device__ __forceinline__ float turn_first(float2 cs, float a, float b) { return fmaf(a, cs.x, -(b * cs.y)); }
__device__ __forceinline__ float turn_second(float2 cs, float a, float b) { return fmaf(a, cs.y, b * cs.x); }

// ---- how a row is shared out among lanes ----------------------------------
// A lane takes two vectors of V elements of one row, at ea and eb, such that
// both elements of every pair it rotates are its own: in the half layout
// vectors c and c + n_dims/2, in the interleaved one (pairs lie inside a
// vector) c and c + head_dim/2; elements past n_dims pass in the same way.
// `lanes` = head_dim / 2V of them hold a row, floor(64 / lanes) rows a wave.
struct RowSplit {
  int lanes;      // per row
  int rows;       // per wave
  uint32_t inv;   // lane / lanes = lane * inv >> 16 for lane < 64
  int head_dim, n_dims, layout;
};
// Whether rows can be split so (the caller takes the general kernel else).
// group: the run of elements that must stay in consecutive lanes (32 for the
// quantised formats' groups, else V).
inline bool row_split(int head_dim, int n_dims, int layout, int v, int group, RowSplit& s) {
  if (head_dim % (2 * v) || head_dim / (2 * v) > 64) return false;
  const bool ok = layout == IT_ROTARY_HALF ? (n_dims / 2) % group == 0 && (head_dim - n_dims) / 2 % group == 0
                                           : (head_dim / 2) % group == 0;
  if (!ok) return false;
  s.lanes = head_dim / (2 * v);
  s.rows = 64 / s.lanes;
  s.inv = uint32_t(65536 / s.lanes + 1);
  s.head_dim = head_dim;
  s.n_dims = n_dims;
  s.layout = layout;
  return true;
}

// Entries of a wave's LDS array of (cos, sin): whole runs of V / 2 pairs.
template <int V>
__host__ __device__ constexpr int angle_room(int n_dims) {
  return (n_dims / 2 + V / 2 - 1) / (V / 2) * (V / 2);
}

// A lane's vectors of its row, and its pairs' (cos, sin) from the wave's LDS
// array of them.
template <int V>
struct LanePairs {
  int ea, eb;       // element offsets in the row
  float2 cs[V];     // half: pairs ea + j; interleaved: j < V/2 pairs ea/2 + j, then eb/2 + j
  __device__ __forceinline__ LanePairs(const RowSplit& s, int c) {
    const int half = s.n_dims >> 1;
    if (s.layout == IT_ROTARY_HALF) {
      const int e = c * V;
      ea = e < half ? e : e + half;
      eb = e < half ? e + half : ea + ((s.head_dim - s.n_dims) >> 1);
    } else {
      ea = c * V;
      eb = ea + (s.head_dim >> 1);
    }
  }
  // From angle_room<V>(n_dims) entries; those of pairs that do not turn are not used.
  __device__ __forceinline__ void load(const RowSplit& s, const float2* all) {
    const int most = angle_room<V>(s.n_dims) - V / 2;
    const int p0 = min(s.layout == IT_ROTARY_HALF ? ea : ea >> 1, most);
    const int p1 = min(s.layout == IT_ROTARY_HALF ? ea + V / 2 : eb >> 1, most);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      cs[j] = all[p0 + j];
      cs[V / 2 + j] = all[p1 + j];
    }
  }
  __device__ __forceinline__ void turn(const RowSplit& s, float (&a)[V], float (&b)[V]) const {
    if (s.layout == IT_ROTARY_HALF) {
      if (ea < (s.n_dims >> 1)) {
#pragma unroll
        for (int j = 0; j < V; ++j) pair(cs[j], a[j], b[j]);
      }
    } else {
      // Pairs past n_dims are left as they are, an infinity among them too.
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        if (ea + 2 * j < s.n_dims) pair(cs[j], a[2 * j], a[2 * j + 1]);
        if (eb + 2 * j < s.n_dims) pair(cs[V / 2 + j], b[2 * j], b[2 * j + 1]);
      }
    }
  }
  static __device__ __forceinline__ void pair(float2 cs, float& a, float& b) {
    const float x = a;
    a = turn_first(cs, x, b);
    b = turn_second(cs, x, b);
  }
};

// The wave's angles of position `pos` into its LDS array: one pair a lane, so
// that the pairs are computed once per wave and not once per row of it.
__device__ __forceinline__ void wave_angles(float2* all, const double* turns, int pairs, int pos, float magnitude, bool transpose,
                                            int lane) {
  for (int p = lane; p < pairs; p += 64) {
    const float2 cs = rotary_angle(turns[p], pos);
    all[p] = make_float2(cs.x * magnitude, transpose ? -cs.y * magnitude : cs.y * magnitude);
  }
  wave_lds_fence();
}

}  // namespace itkv
