// it_beam.hip -- beam search: the best continuations over a group's beams and
// the vocabulary, and per-beam states put in the selected order.
//
//   v[b, i] = score_b + log_softmax(z_b)_i = (score_b - log sum_j exp(z_bj - m_b)) + (z_bi - m_b),
//
// m_b the row's maximum, the n_out largest of a group.  The sum of exponentials is between 1 and
// the vocabulary, so its logarithm is added to the score; added to a maximum near the type's
// largest or lowest value it would vanish, and the score with it.
//
// Two launches.  The first cuts each row into slices of 16 tokens a thread, which
// stay in registers: a slice's maximum, its sum of exponentials against it and its
// n_out best tokens.  The second joins a group's slices: the rows' logarithms,
// then the best of all slices' candidates.
//   The n-th best of a set is bounded from below by the n-th largest of the maxima
// of 64 groups of it, which a wave finds bit by bit; what is not below it (about
// n, up to ties) is listed, and a listed entry's place is the number of listed ones
// before it.  A list that ties overflow is replaced by n rounds of the next best.
//   Times, both launches: four beams of 32000 fp32 logits 10.5 us, 32 groups of eight of
// 100003 bf16 39 (104 and 105 as first written: fp64 throughout, unaligned rows by elements,
// coefficients moved for every token).
//   Sums are in fp64: the order of two beams' candidates hangs on the difference of
// their logarithms, whose fp32 error would decide about as many cases as it has
// units between neighbouring values.
#include <hip/hip_runtime.h>

#include <cmath>

#include "it_internal.hpp"
#include "it_rows.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kPer = 16;                    // tokens a thread holds
constexpr int kSlice = kThreads * kPer;
constexpr int kMaxVocab = 1 << 18;
constexpr int kMaxBeams = 64;
constexpr int kMaxOut = 64;                 // one wave's lanes bound the last place
constexpr int kRoom = 1024;                 // listed entries
constexpr uint32_t kDeadKey = 0x007FFFFFu;  // order_key(-inf)
constexpr int kIndexBits = 18;
static_assert(kMaxVocab <= 1 << kIndexBits, "a token's index in its key");
constexpr int kKeyBits = 32 + kIndexBits;
constexpr uint64_t kKeyMask = (uint64_t(1) << kKeyBits) - 1;

struct SliceSum {
  float top;   // -inf: nothing above it
  float pad;
  double sum;  // of exp(z - top), each off by less than 2^-38 of it, added in fp64
};
struct SelectArgs {
  const char* logits;
  int64_t row_bytes;
  const float* scores;
  float* out_scores;
  int32_t* parents;
  int32_t* tokens;
  SliceSum* sums;     // [rows][slices]
  uint64_t* best;     // [rows][slices][n]: keys of the slice's best, descending; 0: none
  int vocab, slices, n_beams, n_out;
};

// fp32 values as integers of the same order; NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t u = __float_as_uint((z == z ? z : -INFINITY) + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }
// A token's place in its row: larger is earlier, unique, never 0 (a token that is NaN or
// -inf has none).
__device__ __forceinline__ uint64_t token_key(float z, int index) {
  return (uint64_t(order_key(z)) << kIndexBits) | uint32_t(kMaxVocab - 1 - index);
}
__device__ __forceinline__ float token_value(uint64_t k) { return key_value(uint32_t(k >> kIndexBits)); }
__device__ __forceinline__ int token_index(uint64_t k) { return kMaxVocab - 1 - int(k & (kMaxVocab - 1)); }
// fp64 values likewise.
__device__ __forceinline__ uint64_t value_key(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
  return (u >> 63) ? ~u : u | uint64_t(1) << 63;
}
__device__ __forceinline__ double key_double(uint64_t k) {
  return __builtin_bit_cast(double, (k >> 63) ? k & ~(uint64_t(1) << 63) : ~k);
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t x) {
  const int hi = __builtin_amdgcn_update_dpp(0, int(x >> 32), CTRL, 0xF, 0xF, true);
  return uint64_t(uint32_t(hi)) << 32 | uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, 0xF, 0xF, true));
}
// The largest of aligned groups of eight lanes, in each of them.
__device__ __forceinline__ uint64_t eight_max(uint64_t x) {
  x = max(x, dpp64<kDppQuadXor1>(x));
  x = max(x, dpp64<kDppQuadXor2>(x));
  return max(x, dpp64<kDppHalfMirror>(x));
}
__device__ __forceinline__ uint64_t lane64(uint64_t x, int lane) {
  return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(x >> 32), lane))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(x), lane));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
  x = eight_max(x);
  x = max(x, dpp64<kDppRowRor8>(x));
  return max(max(lane64(x, 0), lane64(x, 16)), max(lane64(x, 32), lane64(x, 48)));
}
// The first kBoundBits bits of the n-th largest of the wave's values: a lower bound of it
// (0 where fewer than n are above 0).  Fewer bits let a few more entries through.
constexpr int kBoundBits = 20;
__device__ __forceinline__ uint32_t wave_bound(uint32_t x, int n) {
  uint32_t k = 0u;
#pragma unroll
  for (int b = 31; b >= 32 - kBoundBits; --b) {
    const uint32_t with = k | 1u << b;
    if (__popcll(__ballot(x >= with)) >= n) k = with;
  }
  return k;
}
__device__ __forceinline__ uint32_t eight_max(uint32_t x) {
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppQuadXor1, 0xF, 0xF, true)));
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppQuadXor2, 0xF, 0xF, true)));
  return max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppHalfMirror, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = eight_max(x);
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppRowRor8, 0xF, 0xF, true)));
  const auto at = [&](int lane) { return uint32_t(__builtin_amdgcn_readlane(int(x), lane)); };
  return max(max(at(0), at(16)), max(at(32), at(48)));
}
// The sum over the wave, the same in all lanes.
__device__ __forceinline__ double wave_sum(double x) {
  const auto add = [](double v, auto dpp) { return v + __builtin_bit_cast(double, dpp(__builtin_bit_cast(uint64_t, v))); };
  x = add(x, [](uint64_t v) { return dpp64<kDppQuadXor1>(v); });
  x = add(x, [](uint64_t v) { return dpp64<kDppQuadXor2>(v); });
  x = add(x, [](uint64_t v) { return dpp64<kDppHalfMirror>(v); });
  x = add(x, [](uint64_t v) { return dpp64<kDppRowRor8>(v); });
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const auto at = [&](int lane) { return __builtin_bit_cast(double, lane64(u, lane)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// exp(d) for d <= 0 (an fp64 difference; NaN and -inf give next to nothing, 2^-512): 2^n (1 +
// f h(f)), n the nearest integer to d / ln 2 and h the polynomial through (2^f - 1) / f at
// the eight Chebyshev nodes of [-1/2, 1/2], off by less than 2^-38 of exp(d), and exactly 1 at
// d = 0.  Whole numbers from the low word of a sum with 1.5 x 2^52, exponents as integers.
constexpr double kExp2[8] = {0x1.62e42fef9cc69p-1,  0x1.ebfbdff82a734p-3,  0x1.c6b08da70cce3p-5,  0x1.3b2ab70ad2565p-7,
                             0x1.5d877598350dep-10, 0x1.4308c7183d6a2p-13, 0x1.00c0e4e15189cp-16, 0x1.63b2d7971923fp-20};
// The coefficients stay in scalar registers: as literals each would be moved to a vector
// register again for every token, a third of the work.
struct ExpBelow {
  double c[8], log2e = 1.4426950408889634, least = -354.0, whole = 0x1.8p52;
  __device__ __forceinline__ ExpBelow() {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = kExp2[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("" : "+s"(c[i]));
    asm("" : "+s"(log2e), "+s"(least), "+v"(whole));
  }
  __device__ __forceinline__ double operator()(double d) const {
    d = fmax(d, least);  // of NaN too
    const double n = fma(d, log2e, whole), f = fma(d, log2e, whole - n);
    double h = c[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) h = fma(h, f, c[i]);
    const double m = fma(h, f, 1.0);
    return __hiloint2double(int(uint32_t(__double2hiint(m)) + (uint32_t(__double2loint(n)) << 20)), __double2loint(m));
  }
};

struct Listed {
  uint64_t key, tie;  // the larger key first, of equal keys the smaller tie
};
struct TopShared {
  uint32_t group[64];  // what bounds the n-th best: the largest first words of 64 groups of entries
  Listed list[kRoom];
  uint64_t round[kWaves], round_tie[kWaves];
  uint32_t n;
};
__device__ __forceinline__ bool before(const Listed& a, const Listed& b) { return a.key > b.key || (a.key == b.key && a.tie < b.tie); }

// The n first of the block's entries.  pass(add): calls add(key, tie) for the thread's entries
// that are not below the bound; each(f): f(key, tie) for all of them (key 0: none; no two
// alike), the same ones each time.  put(place, entry): called by one thread for each place
// that an entry takes.  s.n is 0 at the start.
template <class Pass, class Each, class Put>
__device__ __forceinline__ void top_of_block(TopShared& s, int n, Pass&& pass, Each&& each, Put&& put) {
  const int tid = int(threadIdx.x), lane = tid & 63;
  pass([&](uint64_t key, uint64_t tie) {
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kRoom) s.list[at] = {key, tie};
  });
  __syncthreads();
  const uint32_t listed = s.n;
  if (listed <= kRoom) {
    for (uint32_t i = tid; i < listed; i += kThreads) {
      const Listed mine = s.list[i];
      int place = 0;
#pragma unroll 4
      for (uint32_t j = 0; j < listed; ++j) place += before(s.list[j], mine);
      if (place < n) put(place, mine);
    }
    return;
  }
  // More than the list holds are as good as the bound: one place after another.
  Listed last = {~uint64_t(0), 0u};
  bool first = true;
  for (int place = 0; place < n; ++place) {
    Listed mine = {0u, ~uint64_t(0)};
    each([&](uint64_t key, uint64_t tie) {
      const Listed x = {key, tie};
      if (key && (first || before(last, x)) && before(x, mine)) mine = x;
    });
    const uint64_t key = wave_max(mine.key), tie = ~wave_max(mine.key == key ? ~mine.tie : uint64_t(0));
    __syncthreads();  // the round before is read
    if (lane == 0) s.round[tid >> 6] = key, s.round_tie[tid >> 6] = tie;
    __syncthreads();
    Listed best = {0u, ~uint64_t(0)};
    for (int w = 0; w < kWaves; ++w) {
      const Listed x = {s.round[w], s.round_tie[w]};
      if (before(x, best)) best = x;
    }
    if (best.key == 0u) return;  // uniform
    if (mine.key == best.key && mine.tie == best.tie) put(place, mine);
    last = best;
    first = false;
  }
}

// grid: (slice, row).  Bound by the vector units: about 29 operations a token, 16 of them in
// fp64 (32 groups x 8 beams x 100003 bf16 31 us, of which the logits' 51 MB take 8).
template <int DT>
__global__ __launch_bounds__(kThreads, 8) void beam_slices(SelectArgs a) {
  constexpr int es = DT == IT_F32 ? 4 : 2, V = 16 / es, kVecs = kPer / V;
  using In = RowVec<DT, V>;
  __shared__ TopShared top;
  __shared__ double sums[kWaves];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, slice = int(blockIdx.x);
  const int64_t row = blockIdx.y;
  const char* const data = a.logits + row * a.row_bytes;
  const int lo = slice * kSlice, hi = min(a.vocab, lo + kSlice);
  // Thread t's tokens: vectors t, t + 512, .. of the slice, -inf past its end.
  float z[kPer];
  // Rows of an odd vocabulary start anywhere: loads of 16 bytes at an element's alignment.
  typedef typename In::raw Any __attribute__((aligned(es)));
  const Any* const vecs = reinterpret_cast<const Any*>(data + int64_t(lo) * es) + tid;
  if (hi - lo == kSlice) {  // uniform
    typename In::raw w[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) w[j] = __builtin_nontemporal_load(vecs + j * kThreads);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      float f[V];
      In::widen(w[j], f);
#pragma unroll
      for (int e = 0; e < V; ++e) z[j * V + e] = f[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int i = lo + (j * kThreads + tid) * V;
      float f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = -INFINITY;
      if (i + V <= hi) {
        const typename In::raw w = vecs[j * kThreads];
        In::widen(w, f);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < hi) f[e] = load_element(data, i + e, DT);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) z[j * V + e] = f[e];
    }
  }
  float m = -INFINITY;  // NaN does not enter
#pragma unroll
  for (int e = 0; e < kPer; ++e) m = fmaxf(m, z[e]);
  const uint32_t group = eight_max(order_key(m));
  if ((lane & 7) == 0) top.group[tid >> 3] = group;
  if (tid == 0) top.n = 0u;
  uint64_t* const best = a.best + (row * a.slices + slice) * a.n_out;
  if (tid < a.n_out) best[tid] = 0u;
  __syncthreads();
  const uint32_t groups = top.group[lane];  // every wave for itself
  m = key_value(wave_max(groups));
  double sum = 0.0;
  if (m == INFINITY) {  // uniform, as is the other: the tokens there share the row
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += z[e] == m ? 1.0 : 0.0;
  } else if (m > -INFINITY) {
    const ExpBelow exp_below;
    const double top_value = double(m);
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += exp_below(double(z[e]) - top_value);
  }
  sum = wave_sum(sum);
  if (lane == 0) sums[wave] = sum;
  const float least = fmaxf(key_value(max(wave_bound(groups, a.n_out), kDeadKey)), -3.402823466e38f);
  const auto index = [&](int e) { return lo + (e / V * kThreads + tid) * V + e % V; };
  top_of_block(
      top, a.n_out,
      [&](auto&& add) {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (z[e] >= least) add(token_key(z[e], index(e)), uint64_t(0));
      },
      [&](auto&& f) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) f(z[e] > -INFINITY ? token_key(z[e], index(e)) : uint64_t(0), uint64_t(0));
      },
      [&](int place, const Listed& x) { best[place] = x.key; });
  if (tid == 0) {  // past a barrier
    double total = 0.0;
    for (int w = 0; w < kWaves; ++w) total += sums[w];
    a.sums[row * a.slices + slice] = {m, 0.0f, total};
  }
}

// grid: group.  Bound by latency.
__global__ __launch_bounds__(kThreads) void beam_join(SelectArgs a) {
  constexpr int kHeld = 4;  // entries that a thread keeps; more are read again
  __shared__ TopShared top;
  __shared__ double base[kMaxBeams];
  __shared__ float row_top[kMaxBeams];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int64_t g = blockIdx.x, row0 = g * a.n_beams;
  const int per = a.slices * a.n_out, total = a.n_beams * per;
  const uint64_t* const best = a.best + row0 * per;
  // The entries, on their way while the rows' logarithms are taken.
  uint64_t held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = j * kThreads + tid < total ? best[j * kThreads + tid] : 0u;
  static_assert(kMaxVocab / kSlice <= 64, "a row's slices in one wave");
  const ExpBelow exp_below;
  for (int b = wave; b < a.n_beams; b += kWaves) {  // a wave per row, a lane per slice
    SliceSum s = {-INFINITY, 0.0f, 0.0};
    if (lane < a.slices) s = a.sums[(row0 + b) * a.slices + lane];
    const float score = a.scores[g * a.n_beams + b];
    const float m = group_max<64>(s.top);
    const double sum = wave_sum(s.top > -INFINITY ? s.sum * (s.top == m ? 1.0 : exp_below(double(s.top) - double(m))) : 0.0);
    if (lane == 0) {
      // A row at +inf: its tokens there share it equally, log 1/count.
      base[b] = m > -INFINITY && score > -INFINITY ? double(score) - log(sum) : -INFINITY;
      row_top[b] = m;
    }
  }
  const int64_t out = g * a.n_out;
  if (tid < a.n_out) {
    a.out_scores[out + tid] = -INFINITY;
    a.parents[out + tid] = a.tokens[out + tid] = -1;
  }
  if (tid == 0) top.n = 0u;
  __syncthreads();
  const auto entry = [&](int i, uint64_t k, auto&& f) {
    if (k == 0u) return;
    const int b = i / per;
    const float z = token_value(k);
    if (!(base[b] > -INFINITY) || (row_top[b] == INFINITY && z < INFINITY)) return;
    f(value_key(base[b] + (z == INFINITY ? 0.0 : double(z) - double(row_top[b]))), uint64_t(b) << kKeyBits | (kKeyMask - k));
  };
  const auto each = [&](auto&& f) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) entry(j * kThreads + tid, held[j], f);
    for (int i = kHeld * kThreads + tid; i < total; i += kThreads) entry(i, best[i], f);
  };
  uint32_t most = 0u;
  each([&](uint64_t key, uint64_t) { most = max(most, uint32_t(key >> 32)); });
  most = eight_max(most);
  if ((lane & 7) == 0) top.group[tid >> 3] = most;
  __syncthreads();
  const uint32_t least = wave_bound(top.group[lane], a.n_out);
  top_of_block(
      top, a.n_out,
      [&](auto&& add) {
        each([&](uint64_t key, uint64_t tie) {
          if (uint32_t(key >> 32) >= least) add(key, tie);
        });
      },
      each,
      [&](int place, const Listed& x) {
        a.out_scores[out + place] = float(key_double(x.key));
        a.parents[out + place] = int32_t(x.tie >> kKeyBits);
        a.tokens[out + place] = token_index(kKeyMask - (x.tie & kKeyMask));
      });
}

// ---- per-beam states -------------------------------------------------------
// A thread holds one unit of U's size of all of a group's rows: every row that
// changes is read, then written, so no second buffer and no order is needed.
// Bound by memory: a changed row is written once, its parent read once (from a
// cache where several continue it).  grid: (units, group, outer).
// Large workgroups, as few as possible, and stores that do not stay in L2: 8 groups of 8 rows
// of 256 KB in 28 arrays (470 MB, 7 of 8 rows replaced) 137 to 146 us with 1024 threads, 186 with
// 512, 178 to 180 with 256; with stores that stay 143 to 151 and, with 256 threads, 181 to 188.
template <class U, int K, int B>
__global__ __launch_bounds__(B) void beam_rows(char* x, int64_t units, int64_t row_stride, int64_t outer_stride, int n_beams,
                                               const int32_t* parents) {
  const int64_t u = int64_t(blockIdx.x) * B + threadIdx.x;
  if (u >= units) return;
  const int g = int(blockIdx.y);
  char* const base = x + int64_t(blockIdx.z) * outer_stride + int64_t(g) * n_beams * row_stride + u * int64_t(sizeof(U));
  const int32_t* const from = parents + int64_t(g) * n_beams;
  U v[K];
  int p[K];
#pragma unroll
  for (int j = 0; j < K; ++j) p[j] = from[min(j, n_beams - 1)];
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j >= n_beams || p[j] < 0 || p[j] >= n_beams || p[j] == j) p[j] = -1;  // stays
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (p[j] >= 0) v[j] = *reinterpret_cast<const U*>(base + p[j] * row_stride);
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (p[j] >= 0) __builtin_nontemporal_store(v[j], reinterpret_cast<U*>(base + j * row_stride));
}

template <class U, int K, int B>
void launch_beams(char* x, int64_t units, int64_t row_stride, int64_t outer_stride, int n_outer, int n_groups, int n_beams,
                  const int32_t* parents, hipStream_t s) {
  const dim3 grid(unsigned((units + B - 1) / B), unsigned(n_groups), unsigned(n_outer));
  hipLaunchKernelGGL((beam_rows<U, K, B>), grid, dim3(B), 0, s, x, units, row_stride, outer_stride, n_beams, parents);
}
template <class U>
void launch_rows(char* x, int64_t units, int64_t row_stride, int64_t outer_stride, int n_outer, int n_groups, int n_beams,
                 const int32_t* parents, hipStream_t s) {
  // 64 rows of 16 bytes are 256 registers: fewer threads where there are more rows.  Short rows
  // of few groups are spread over more workgroups.
  const bool large = units >= 4096;
#define IT_BEAMS(K, B) launch_beams<U, K, B>(x, units, row_stride, outer_stride, n_outer, n_groups, n_beams, parents, s)
  if (n_beams <= 4) large ? IT_BEAMS(4, 1024) : IT_BEAMS(4, 256);
  else if (n_beams <= 8) large ? IT_BEAMS(8, 1024) : IT_BEAMS(8, 256);
  else if (n_beams <= 16) large ? IT_BEAMS(16, 1024) : IT_BEAMS(16, 256);
  else if (n_beams <= 32) large ? IT_BEAMS(32, 512) : IT_BEAMS(32, 256);
  else IT_BEAMS(64, 256);
#undef IT_BEAMS
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }
int slices_of(int32_t vocab) { return (vocab + kSlice - 1) / kSlice; }
bool sizes_ok(const char* who, int32_t n_groups, int32_t n_beams, int32_t vocab, int32_t n_out) {
  if (n_groups < 0 || n_beams < 1 || n_beams > kMaxBeams || int64_t(n_groups) * n_beams > 65535 || vocab < 1 || vocab > kMaxVocab ||
      n_out < 1 || n_out > kMaxOut) {
    fail(IT_INVALID_INPUT, "%s: n_groups %d, n_beams %d (1 to %d; to 65535 rows), vocab %d (1 to %d), n_out %d (1 to %d)", who, n_groups,
         n_beams, kMaxBeams, vocab, kMaxVocab, n_out, kMaxOut);
    return false;
  }
  return true;
}
}  // namespace

extern "C" size_t it_beam_select_workspace(int32_t n_groups, int32_t n_beams, int32_t vocab, int32_t n_out) {
  if (!sizes_ok("it_beam_select_workspace", n_groups, n_beams, vocab, n_out)) return 0;
  const size_t slices = size_t(n_groups) * size_t(n_beams) * size_t(slices_of(vocab));
  return align256(slices * sizeof(SliceSum)) + align256(slices * size_t(n_out) * 8);
}

extern "C" int32_t it_beam_select(const void* logits, int32_t dtype, int64_t row_stride, int32_t n_groups, int32_t n_beams, int32_t vocab,
                                  const float* scores, int32_t n_out, float* out_scores, int32_t* parents, int32_t* tokens, void* ws,
                                  size_t ws_bytes, void* stream) {
  const char* who = "it_beam_select";
  if (dtype != IT_F32 && dtype != IT_F16 && dtype != IT_BF16) return fail(IT_NOT_IMPLEMENTED, "%s: dtype %d (F32, F16 or BF16)", who, dtype);
  if (!sizes_ok(who, n_groups, n_beams, vocab, n_out)) return IT_INVALID_INPUT;
  if (n_groups == 0) return IT_OK;
  if (int64_t(n_groups) * n_beams > 1 && (row_stride < vocab || row_stride > int64_t(1) << 40))
    return fail(IT_INVALID_INPUT, "%s: row_stride %lld below vocab %d (or above 2^40)", who, (long long)row_stride, vocab);
  if (!logits || !scores || !out_scores || !parents || !tokens) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  const int64_t es = dtype_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(logits) % uintptr_t(es)) return fail(IT_INVALID_INPUT, "%s: logits must be aligned to their elements", who);
  const size_t need = it_beam_select_workspace(n_groups, n_beams, vocab, n_out);
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(IT_INVALID_INPUT, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", who, ws ? ws_bytes : size_t(0), need);
  SelectArgs a{};
  a.logits = static_cast<const char*>(logits);
  a.row_bytes = row_stride * es;
  a.scores = scores;
  a.out_scores = out_scores;
  a.parents = parents;
  a.tokens = tokens;
  a.vocab = vocab;
  a.slices = slices_of(vocab);
  a.n_beams = n_beams;
  a.n_out = n_out;
  a.sums = static_cast<SliceSum*>(ws);
  a.best = reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + align256(size_t(n_groups) * size_t(n_beams) * size_t(a.slices) * sizeof(SliceSum)));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(unsigned(a.slices), unsigned(n_groups * n_beams));
  switch (dtype) {
    case IT_F32: hipLaunchKernelGGL(beam_slices<IT_F32>, grid, dim3(kThreads), 0, s, a); break;
    case IT_BF16: hipLaunchKernelGGL(beam_slices<IT_BF16>, grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(beam_slices<IT_F16>, grid, dim3(kThreads), 0, s, a); break;
  }
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) {
    hipLaunchKernelGGL(beam_join, dim3(unsigned(n_groups)), dim3(kThreads), 0, s, a);
    e = hipGetLastError();
  }
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}

extern "C" int32_t it_beam_reorder(void* x, int64_t row_bytes, int64_t row_stride, int32_t n_outer, int64_t outer_stride, int32_t n_groups,
                                   int32_t n_beams, const int32_t* parents, void* stream) {
  const char* who = "it_beam_reorder";
  const int64_t kFar = int64_t(1) << 40;
  if (n_groups < 0 || n_groups > 65535 || n_beams < 1 || n_beams > kMaxBeams || n_outer < 0 || n_outer > 65535 || row_bytes < 0 || row_bytes > kFar)
    return fail(IT_INVALID_INPUT, "%s: row_bytes %lld, n_outer %d, n_groups %d (to 65535), n_beams %d (1 to %d)", who, (long long)row_bytes,
                n_outer, n_groups, n_beams, kMaxBeams);
  const int64_t rows = int64_t(n_groups) * n_beams;
  if (rows > 1 && (row_stride < row_bytes || row_stride > kFar))
    return fail(IT_INVALID_INPUT, "%s: row_stride %lld below row_bytes %lld (or above 2^40)", who, (long long)row_stride, (long long)row_bytes);
  if (n_outer > 1 && (outer_stride < (rows - 1) * row_stride + row_bytes || outer_stride > kFar))
    return fail(IT_INVALID_INPUT, "%s: outer_stride %lld below an array of %lld rows", who, (long long)outer_stride, (long long)rows);
  if (rows == 0 || n_outer == 0 || row_bytes == 0) return IT_OK;
  if (!x || !parents) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  if (reinterpret_cast<uintptr_t>(parents) & 3u) return fail(IT_INVALID_INPUT, "%s: parents must be aligned to 4 bytes", who);
  if (rows == 1) row_stride = 0;
  if (n_outer == 1) outer_stride = 0;
  const uintptr_t first = reinterpret_cast<uintptr_t>(x), at = reinterpret_cast<uintptr_t>(parents);
  const int64_t span = (n_outer - 1) * outer_stride + (rows - 1) * row_stride + row_bytes;
  if (at < first + uintptr_t(span) && first < at + uintptr_t(rows) * 4) return fail(IT_INVALID_INPUT, "%s: parents lie inside x", who);
  const uintptr_t all = first | uintptr_t(row_bytes) | uintptr_t(row_stride) | uintptr_t(outer_stride);
  const int unit = (all & 15u) == 0 ? 16 : (all & 3u) == 0 ? 4 : 1;
  if (row_bytes / unit > int64_t(1) << 31) return fail(IT_INVALID_INPUT, "%s: rows of %lld bytes", who, (long long)row_bytes);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* const p = static_cast<char*>(x);
  if (unit == 16) launch_rows<u32x4>(p, row_bytes / 16, row_stride, outer_stride, n_outer, n_groups, n_beams, parents, s);
  else if (unit == 4) launch_rows<uint32_t>(p, row_bytes / 4, row_stride, outer_stride, n_outer, n_groups, n_beams, parents, s);
  else launch_rows<uint8_t>(p, row_bytes, row_stride, outer_stride, n_outer, n_groups, n_beams, parents, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
