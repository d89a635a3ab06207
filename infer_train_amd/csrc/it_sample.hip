// it_sample.hip -- one token per row of logits: temperature, min-p, top-k,
// top-p and a given uniform number.
//
//   w_i = exp((z_i - max z) / T) in the order (z descending, index ascending);
//   every filter keeps a prefix of that order, so the kept set is a length n,
//   and the token is the first i with w_0 + .. + w_i > u (w_0 + .. + w_{n-1}).
//
// So nothing has to be sorted: each filter's end and the draw are one question,
// "where along the order does the count, or the mass, reach X?", answered by a
// histogram over the order and a second, finer one inside the bin it names.
// Masses are 64-bit integers (2^-44 of the largest weight): their sums are
// exact, so any number of workgroups may add them in any order, and the same
// row gives the same token in any batch.
//
// Two launches.  The first reads the logits from HBM and takes each slice's
// maximum.  The second reads them again (from the last-level cache where the
// call's logits fit its 256 MB), weighs them in fp64 against the row's maximum
// and adds counts and masses of 1024 bins, linear in z, in LDS and then per row;
// the row's last workgroup to finish answers the questions.  Where top-k or
// min-p bound the tokens that matter, those alone are weighed, and listed, so
// that the last workgroup need not read the row a third time: of the maxima of
// groups of tokens the k-th largest is a lower bound of the k-th largest token.
#include <hip/hip_runtime.h>

#include <cmath>

#include "it_rotary.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2 * kThreads;  // locate(): two per thread
constexpr int kList = 2048;          // tokens listed per row, and held in LDS
constexpr int kMaxSlices = 32;
constexpr int kGroups = 2 * kWaves;  // group maxima per slice: half waves
constexpr int kMaxVocab = 1 << 18;   // a sum of weights stays below 2^62
constexpr int kIndexBits = 18;
constexpr double kUnit = 0x1p44;      // weight of the largest token
constexpr double kBinsPerBit = 22.0;  // of log2 weight; 45.x bits weigh at all
constexpr uint32_t kDeadKey = 0x007FFFFFu;  // order_key(-inf)

struct RowState {
  uint32_t ticket, n_list;
  uint64_t pad[31];
  uint64_t best[kMaxSlices];               // order of each slice's first token, 0: nothing above -inf
  uint32_t group_max[kMaxSlices * kGroups];
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t list[kList];
};
static_assert(sizeof(RowState) % 256 == 0, "rows of the workspace stay aligned");

struct SampleArgs {
  const char* logits;
  int64_t row_bytes;
  const float *u, *temperatures, *top_ps, *min_ps;
  const int32_t* top_ks;
  int32_t* tokens;
  float* probs;
  RowState* rows;
  int vocab, slices;
  float temperature, top_p, min_p;
  int top_k;
};

// fp32 values as integers of the same order; NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t u = __float_as_uint((z == z ? z : -INFINITY) + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }
// A token's place in the order: larger is earlier; unique in a row.
__device__ __forceinline__ uint64_t order_of(float z, int index) {
  return (uint64_t(order_key(z)) << kIndexBits) | uint32_t(kMaxVocab - 1 - index);
}
__device__ __forceinline__ float order_value(uint64_t o) { return key_value(uint32_t(o >> kIndexBits)); }
__device__ __forceinline__ int order_index(uint64_t o) { return kMaxVocab - 1 - int(o & (kMaxVocab - 1)); }

// 2^x for x in [-46, 0] within 2^-51 of its value: the Taylor sum of exp(f ln 2)
// around the nearest integer, |f| <= 1/2, to f^12 (the next term is below 2^-58).
__device__ __forceinline__ double exp2_neg(double x) {
  const double n = __builtin_rint(x), f = (x - n) * 0.6931471805599453;
  double p = 1.0 / 479001600.0;
  constexpr double kInv[12] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                               1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800};
#pragma unroll
  for (int i = 11; i >= 0; --i) p = fma(p, f, kInv[i]);
  return __builtin_amdgcn_ldexp(p, int(n));
}

// A row's settings, the same in all its threads.
struct Weigher {
  float top;      // max z
  float floor;    // tokens below weigh nothing, fail min-p or cannot be among the first k
  double bits;    // log2(e) / T
  double min_p;
  // Weight and bin of a token with z >= floor; false: not kept.
  __device__ __forceinline__ bool operator()(float z, uint64_t& w, int& bin) const {
    const double x = z == top ? 0.0 : (double(z) - double(top)) * bits;
    if (!(x > -46.0)) return false;
    const double e = exp2_neg(x);
    // Rounded to a whole number of units by the sum with 2^52.
    w = __builtin_bit_cast(uint64_t, fma(e, kUnit, 0x1p52)) & ((uint64_t(1) << 52) - 1);
    bin = int(x * -kBinsPerBit);
    return w != 0 && e >= min_p;
  }
};

// f(index, z) for tokens of a row, 16-byte vectors `lo` .. `hi` of its aligned
// part, with `head` also the tokens before it and with `tail` those behind.
template <int DT, class F>
__device__ __forceinline__ void each_token(const char* row, int vocab, int slice, int slices, F&& f) {
  constexpr int es = DT == IT_F32 ? 4 : 2, V = 16 / es, U = 4;
  using In = RowVec<DT, V>;
  const int tid = int(threadIdx.x);
  const int head = min(vocab, int((16 - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / es);
  const int vecs = (vocab - head) / V, done = head + vecs * V;
  const int per = (vecs + slices - 1) / slices, lo = min(vecs, slice * per), hi = min(vecs, lo + per);
  if (slice == 0 && tid < head) f(tid, load_element(row, tid, DT));
  const auto* const v = reinterpret_cast<const typename In::raw*>(row + head * es);
  for (int x0 = lo + tid; x0 < hi; x0 += kThreads * U) {
    typename In::raw w[U];
#pragma unroll
    for (int j = 0; j < U; ++j) w[j] = v[min(x0 + j * kThreads, hi - 1)];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int x = x0 + j * kThreads;
      if (x >= hi) break;
      float z[V];
      In::widen(w[j], z);
#pragma unroll
      for (int e = 0; e < V; ++e) f(head + x * V + e, z[e]);
    }
  }
  if (slice == slices - 1 && tid < vocab - done) f(done + tid, load_element(row, done + tid, DT));
}

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int lane) { return uint64_t(__shfl((unsigned long long)(x), lane)); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint64_t y = uint64_t(__shfl_xor((unsigned long long)(x), o));
    x = y > x ? y : x;
  }
  return x;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_maxima(SampleArgs a) {
  __shared__ uint64_t best_of[kWaves];
  const int slice = int(blockIdx.x), lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6);
  RowState& rs = a.rows[blockIdx.y];
  // Clear what the second launch adds to.
  if (slice == 0 && threadIdx.x == 0) rs.ticket = rs.n_list = 0u;
  for (int b = slice * kThreads + int(threadIdx.x); b < kBins; b += a.slices * kThreads) rs.count[b] = 0u, rs.mass[b] = 0u;
  float top = -INFINITY;
  int at = -1;
  each_token<DT>(a.logits + int64_t(blockIdx.y) * a.row_bytes, a.vocab, slice, a.slices, [&](int i, float z) {
    if (z > top) top = z, at = i;  // the first of equals: a thread's tokens come in ascending order
  });
  uint64_t best = at < 0 ? 0u : order_of(top, at);
  uint32_t group = order_key(top);
#pragma unroll
  for (int o = 16; o; o >>= 1) group = max(group, uint32_t(__shfl_xor(int(group), o)));
  if ((lane & 31) == 0) rs.group_max[slice * kGroups + wave * 2 + (lane >> 5)] = group;
  best = wave_max64(best);
  if (lane == 0) best_of[wave] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWaves; ++i) best = best_of[i] > best ? best_of[i] : best;
    rs.best[slice] = best;
  }
}

struct Shared {
  uint64_t mass[kBins];   // the row's bins (before the last workgroup: its slice's)
  uint64_t fine[kBins];   // masses of the bins inside one of them
  uint64_t cand[kList];   // tokens of that bin (before: the slice's list)
  uint64_t last[64];
  uint32_t count[kBins];
  uint32_t fine_count[kBins];
  uint64_t wave_mass[kWaves];
  uint32_t wave_count[kWaves];
  unsigned long long lo, hi;
  uint32_t n, is_last, base;
  // locate()'s and select()'s answers
  uint64_t before_mass, total_mass, mass_to, weight;
  uint32_t before_count, total_count, in_bin, bin;
  int token;
};

// The bin in which the cumulative count (or mass), from before_* on, reaches
// `goal`: s.bin, s.in_bin tokens, what is before it in s.before_*.
__device__ __forceinline__ void locate(Shared& s, const uint32_t* count, const uint64_t* mass, bool by_count, uint64_t goal,
                                       uint32_t before_count, uint64_t before_mass) {
  const int t = int(threadIdx.x), lane = t & 63, wave = t >> 6;
  const uint32_t c0 = count[2 * t], c1 = count[2 * t + 1];
  const uint64_t m0 = mass[2 * t], m1 = mass[2 * t + 1];
  uint32_t c = c0 + c1;
  uint64_t m = m0 + m1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t cu = uint32_t(__shfl_up(int(c), o));
    const uint64_t mu = uint64_t(__shfl_up((unsigned long long)(m), o));
    if (lane >= o) c += cu, m += mu;
  }
  if (lane == 63) s.wave_count[wave] = c, s.wave_mass[wave] = m;
  __syncthreads();
  uint32_t cs = before_count + c - c0 - c1;
  uint64_t ms = before_mass + m - m0 - m1;
  for (int w = 0; w < wave; ++w) cs += s.wave_count[w], ms += s.wave_mass[w];
  if (t == kThreads - 1) s.total_count = cs + c0 + c1, s.total_mass = ms + m0 + m1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t ci = i ? c1 : c0;
    const uint64_t mi = i ? m1 : m0;
    const uint64_t before = by_count ? cs : ms, after = before + (by_count ? uint64_t(ci) : mi);
    if (before < goal && goal <= after) {
      s.bin = uint32_t(2 * t + i);
      s.in_bin = ci;
      s.before_count = cs;
      s.before_mass = ms;
    }
    cs += ci;
    ms += mi;
  }
  __syncthreads();
}

template <int DT>
struct Row {
  const char* data;
  int vocab;
  const uint64_t* list;  // or NULL: too many tokens to list
  uint32_t n_list;
  Weigher weigh;
  // f(order, z) for the row's tokens with lo <= z <= hi that may be kept.
  template <class F>
  __device__ __forceinline__ void each(float lo, float hi, F&& f) const {
    if (list) {
      for (uint32_t i = threadIdx.x; i < n_list; i += kThreads) {
        const uint64_t o = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const float z = order_value(o);
        if (z >= lo && z <= hi) f(o, z);
      }
    } else {
      each_token<DT>(data, vocab, 0, 1, [&](int i, float z) {
        if (z >= lo && z <= hi) f(order_of(z, i), z);
      });
    }
  }
};

// The token at which the cumulative count (or mass) along the order reaches
// `goal`: s.token, its weight, and the mass up to and with it in s.mass_to.
// All threads of the workgroup; 1 <= goal <= the row's total.
template <int DT>
__device__ void select(Shared& s, const Row<DT>& row, bool by_count, uint64_t goal) {
  const int t = int(threadIdx.x);
  locate(s, s.count, s.mass, by_count, goal, 0u, 0u);
  const int bin = int(s.bin);
  uint32_t n = s.in_bin, bc = s.before_count;
  uint64_t bm = s.before_mass;
  // The bin's z, widened by what fp32 and fp64 rounding can move an edge.
  float zlo = row.weigh.floor, zhi = INFINITY;
  if (row.weigh.top < INFINITY && row.weigh.bits > 0.0) {
    const double edge = 1.0 / (kBinsPerBit * row.weigh.bits), top = double(row.weigh.top);
    const double first = top - double(bin) * edge, end = top - double(bin + 1) * edge;
    zhi = float(first + (fabs(first) + edge) * 0x1p-20);
    zlo = fmaxf(zlo, float(end - (fabs(end) + edge) * 0x1p-20));
  }
  bool held = n <= kList;  // in s.cand
  if (t == 0) s.n = 0u, s.lo = ~0ull, s.hi = 0ull;
  __syncthreads();
  unsigned long long tlo = ~0ull, thi = 0ull;
  row.each(zlo, zhi, [&](uint64_t o, float z) {
    uint64_t w;
    int b;
    if (!row.weigh(z, w, b) || b != bin) return;
    tlo = o < tlo ? o : tlo;
    thi = o > thi ? o : thi;
    if (held) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kList) s.cand[at] = o;
    }
  });
  if (thi) {
    atomicMin(&s.lo, tlo);
    atomicMax(&s.hi, thi);
  }
  __syncthreads();
  uint64_t lo = s.lo, hi = s.hi;
  uint32_t cands = min(s.n, uint32_t(kList));
  // f(order) for the tokens with lo <= order <= hi.
  const auto each_in = [&](auto&& f) {
    if (held) {
      for (uint32_t i = t; i < cands; i += kThreads) {
        const uint64_t o = s.cand[i];
        if (o >= lo && o <= hi) f(o);
      }
    } else {
      row.each(order_value(lo), order_value(hi), [&](uint64_t o, float) {
        if (o >= lo && o <= hi) f(o);
      });
    }
  };
  // 1024 bins of a power of two of orders each: nine bits of hi - lo < 2^50 a
  // turn or more, orders are unique.
  for (int turn = 0; n > 64 && turn < 6; ++turn) {
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
    for (int b = t; b < kBins; b += kThreads) s.fine_count[b] = 0u, s.fine[b] = 0u;
    __syncthreads();
    each_in([&](uint64_t o) {
      uint64_t w = 0;
      int b;
      row.weigh(order_value(o), w, b);
      const uint32_t x = uint32_t((hi - o) >> shift);
      atomicAdd(&s.fine_count[x], 1u);
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.fine[x]), (unsigned long long)(w));
    });
    __syncthreads();
    locate(s, s.fine_count, s.fine, by_count, goal, bc, bm);
    n = s.in_bin;
    bc = s.before_count;
    bm = s.before_mass;
    hi -= uint64_t(s.bin) << shift;
    const uint64_t width = uint64_t(1) << shift;
    lo = hi >= width && hi - width + 1 > lo ? hi - width + 1 : lo;
    if (!held && n <= kList) {
      if (t == 0) s.n = 0u;
      __syncthreads();
      each_in([&](uint64_t o) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < kList) s.cand[at] = o;
      });
      __syncthreads();
      held = true;
      cands = min(s.n, uint32_t(kList));
    }
    __syncthreads();
  }
  if (t == 0) s.n = 0u;
  __syncthreads();
  each_in([&](uint64_t o) {
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < 64) s.last[at] = o;
  });
  __syncthreads();
  if (t < 64) {  // one wave: a token a lane, each with the mass of those before it
    n = min(n, 64u);
    const uint64_t own = t < int(n) ? s.last[t] : 0u;
    uint64_t w = 0;
    int b;
    if (t < int(n)) row.weigh(order_value(own), w, b);
    uint32_t ci = 0u;
    uint64_t mi = 0u;
    for (uint32_t j = 0; j < n; ++j) {
      const uint64_t o = shfl64(own, int(j)), wj = shfl64(w, int(j));
      if (o >= own) ci += 1u, mi += wj;
    }
    const uint64_t after = by_count ? uint64_t(bc + ci) : bm + mi, before = by_count ? after - 1 : after - w;
    if (t < int(n) && before < goal && goal <= after) {
      s.token = order_index(own);
      s.weight = w;
      s.mass_to = bm + mi;
    }
  }
  __syncthreads();
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_draw(SampleArgs a) {
  __shared__ Shared s;
  const int t = int(threadIdx.x), lane = t & 63, slice = int(blockIdx.x), row = int(blockIdx.y);
  RowState& rs = a.rows[row];
  const uint64_t best = wave_max64(lane < a.slices ? rs.best[lane] : 0u);
  const float temp = a.temperatures ? a.temperatures[row] : a.temperature;
  if (best == 0u || !(temp > 0.0f)) {  // uniform: an empty row, or the first of the order
    if (slice == 0 && t == 0) {
      a.tokens[row] = best ? order_index(best) : -1;
      if (a.probs) a.probs[row] = best ? 1.0f : 0.0f;
    }
    return;
  }
  const int top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[row] : a.top_p, min_p = a.min_ps ? a.min_ps[row] : a.min_p;
  Weigher weigh;
  weigh.top = order_value(best);
  weigh.bits = 1.4426950408889634 / double(temp);
  weigh.min_p = min_p > 0.0f ? fmin(double(min_p), 1.0) : 0.0;
  // Below floor a weight rounds to nothing or fails min-p: z - top < T ln(max(min_p, 2^-46)),
  // widened by fp32's rounding.
  weigh.floor = weigh.top;
  if (weigh.top < INFINITY) {
    const double low = double(weigh.top) + fmax(log2(fmax(weigh.min_p, 0x1p-46)), -46.0) / weigh.bits;
    weigh.floor = float(low - fabs(low) * 0x1p-20);
  }
  bool listed = weigh.min_p > 0.0;
  const int groups = a.slices * kGroups;
  if (top_k > 0 && top_k <= groups) {
    // The first sixteen bits of the top_k-th largest group maximum: at least
    // top_k tokens have keys that large.
    uint32_t g[kMaxSlices * kGroups / 64], key = 0u;
#pragma unroll
    for (int j = 0; j < kMaxSlices * kGroups / 64; ++j) {
      const int i = j * 64 + lane;
      g[j] = i < groups ? rs.group_max[i] : 0u;
    }
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
      const uint32_t with = key | bit;
      int n = 0;
#pragma unroll
      for (int j = 0; j < kMaxSlices * kGroups / 64; ++j) n += __popcll(__ballot(g[j] >= with));
      if (n >= top_k) key = with;
    }
    if (key > kDeadKey) weigh.floor = fmaxf(weigh.floor, key_value(key));
    listed = true;
  }
  // Whatever the floor, a token at -inf is never kept.
  weigh.floor = fmaxf(weigh.floor, -3.402823466e38f);

  for (int b = t; b < kBins; b += kThreads) s.count[b] = 0u, s.mass[b] = 0u;
  if (t == 0) s.n = 0u;
  __syncthreads();
  const char* const data = a.logits + int64_t(row) * a.row_bytes;
  each_token<DT>(data, a.vocab, slice, a.slices, [&](int i, float z) {
    if (!(z >= weigh.floor)) return;
    uint64_t w;
    int b;
    if (!weigh(z, w, b)) return;
    atomicAdd(&s.count[b], 1u);
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), (unsigned long long)(w));
    if (listed) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kList) s.cand[at] = order_of(z, i);
    }
  });
  __syncthreads();
  for (int b = t; b < kBins; b += kThreads) {
    if (s.count[b] == 0u) continue;
    atomicAdd(&rs.count[b], s.count[b]);
    atomicAdd(reinterpret_cast<unsigned long long*>(&rs.mass[b]), (unsigned long long)(s.mass[b]));
  }
  if (listed) {
    if (t == 0) s.base = atomicAdd(&rs.n_list, min(s.n, uint32_t(kList + 1)));
    __syncthreads();
    if (s.n <= kList && s.base + s.n <= kList)
      for (uint32_t i = t; i < s.n; i += kThreads) rs.list[s.base + i] = s.cand[i];
  }
  // The row's last workgroup: every other one's additions are visible to it.
  __threadfence();
  __syncthreads();
  if (t == 0) s.is_last = atomicAdd(&rs.ticket, 1u) == uint32_t(a.slices - 1);
  __syncthreads();
  if (!s.is_last) return;  // uniform
  __threadfence();
  for (int b = t; b < kBins; b += kThreads) {
    s.count[b] = __hip_atomic_load(&rs.count[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s.mass[b] = __hip_atomic_load(&rs.mass[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const uint32_t n_list = __hip_atomic_load(&rs.n_list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const Row<DT> r{data, a.vocab, listed && n_list <= kList ? rs.list : nullptr, n_list, weigh};
  __syncthreads();
  locate(s, s.count, s.mass, true, 1u, 0u, 0u);  // for the totals
  uint64_t kept = s.total_mass;
  const uint32_t tokens = s.total_count;
  __syncthreads();
  // Where top-k ends, where top-p ends (each leaves the mass kept), the draw.
  for (int question = 0; question < 3; ++question) {
    uint64_t goal;
    if (question == 0) {
      if (top_k <= 0 || uint32_t(top_k) >= tokens) continue;
      goal = uint64_t(top_k);
    } else if (question == 1) {
      if (!(top_p < 1.0f)) continue;  // NaN: off
      // before < top_p kept  <=>  before < ceil(top_p kept), before being whole.
      const double part = top_p > 0.0f ? ceil(double(top_p) * double(kept)) : 0.0;
      goal = part < 1.0 ? 1u : uint64_t(part);
      if (goal >= kept) continue;
    } else {
      const float u = a.u[row];
      const double at = u > 0.0f ? fmin(double(u), 1.0) * double(kept) : 0.0;  // kept <= 2^62
      goal = uint64_t(at);
      goal = (goal < kept ? goal : kept - 1) + 1;
    }
    select(s, r, question == 0, goal);
    if (question < 2) kept = s.mass_to;
    __syncthreads();
  }
  if (t == 0) {
    a.tokens[row] = s.token;
    if (a.probs) a.probs[row] = float(double(s.weight) / double(kept));
  }
}

// Slices of a row: of 4096 tokens or more, as many as leave 2048 workgroups
// (four resident on each of 256 CUs, twice).  The result does not depend on it.
int slice_count(int32_t rows, int32_t vocab) {
  int s = (vocab + 4095) / 4096;
  const int fill = 2048 / rows > 0 ? 2048 / rows : 1;
  s = s < fill ? s : fill;
  return s < kMaxSlices ? s : kMaxSlices;
}

template <int DT>
void launch_sample(const SampleArgs& a, int32_t rows, hipStream_t s) {
  const dim3 grid(unsigned(a.slices), unsigned(rows));
  hipLaunchKernelGGL(sample_maxima<DT>, grid, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(sample_draw<DT>, grid, dim3(kThreads), 0, s, a);
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
}  // namespace

extern "C" size_t it_sample_workspace(int32_t n_rows, int32_t vocab) {
  return n_rows > 0 && vocab > 0 ? size_t(n_rows) * sizeof(RowState) : 0;
}

extern "C" int32_t it_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t n_rows, int32_t vocab, const float* u,
                             const float* temperatures, const int32_t* top_ks, const float* top_ps, const float* min_ps,
                             float temperature, int32_t top_k, float top_p, float min_p, int32_t* tokens, float* probs, void* ws,
                             size_t ws_bytes, void* stream) {
  const char* who = "it_sample";
  if (dtype != IT_F32 && dtype != IT_F16 && dtype != IT_BF16) return fail(IT_NOT_IMPLEMENTED, "%s: dtype %d (F32, F16 or BF16)", who, dtype);
  if (n_rows < 0 || n_rows > 65535) return fail(IT_INVALID_INPUT, "%s: n_rows %d outside [0, 65535]", who, n_rows);
  if (vocab <= 0) return fail(IT_INVALID_INPUT, "%s: vocab %d", who, vocab);
  if (vocab > kMaxVocab) return fail(IT_NOT_IMPLEMENTED, "%s: vocab %d above %d", who, vocab, kMaxVocab);
  if (n_rows > 1 && (row_stride < vocab || row_stride > int64_t(1) << 40))
    return fail(IT_INVALID_INPUT, "%s: row_stride %lld below vocab %d (or above 2^40)", who, (long long)row_stride, vocab);
  if (!temperatures && (!(temperature >= 0.0f) || std::isinf(temperature)))
    return fail(IT_INVALID_INPUT, "%s: temperature %g must be finite, >= 0", who, double(temperature));
  if (!top_ps && std::isnan(top_p)) return fail(IT_INVALID_INPUT, "%s: top_p is NaN", who);
  if (!min_ps && !(min_p <= 1.0f)) return fail(IT_INVALID_INPUT, "%s: min_p %g must be <= 1", who, double(min_p));
  if (n_rows == 0) return IT_OK;
  if (!logits || !u || !tokens) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  const int64_t es = dtype_bytes(dtype);
  if (!aligned(logits, uintptr_t(es))) return fail(IT_INVALID_INPUT, "%s: logits must be aligned to their elements", who);
  if (!ws || ws_bytes < it_sample_workspace(n_rows, vocab) || !aligned(ws, 256))
    return fail(IT_INVALID_INPUT, "%s: workspace of %zu bytes, %zu needed, 256-byte aligned", who, ws ? ws_bytes : size_t(0),
                it_sample_workspace(n_rows, vocab));
  SampleArgs a{};
  a.logits = static_cast<const char*>(logits);
  a.row_bytes = (n_rows > 1 ? row_stride : int64_t(vocab)) * es;
  a.u = u;
  a.temperatures = temperatures;
  a.top_ks = top_ks;
  a.top_ps = top_ps;
  a.min_ps = min_ps;
  a.tokens = tokens;
  a.probs = probs;
  a.rows = static_cast<RowState*>(ws);
  a.vocab = vocab;
  a.slices = slice_count(n_rows, vocab);
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == IT_F32) launch_sample<IT_F32>(a, n_rows, s);
  else if (dtype == IT_F16) launch_sample<IT_F16>(a, n_rows, s);
  else launch_sample<IT_BF16>(a, n_rows, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
