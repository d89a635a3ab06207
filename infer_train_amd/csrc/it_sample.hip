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
// The logits are read from HBM for their maximum and again, from a cache where the
// call's logits fit it, to be weighed in fp64 against that: counts and masses are
// added into 2048 bins, linear in z, in LDS.  Then the few bins that the answers lie
// in are found, their tokens gathered, and the answers taken from those.  Where
// top-k or min-p bound the tokens that matter, those alone are weighed, and listed,
// so that the row need not be read a third time: of the maxima of groups of tokens
// the k-th largest is a lower bound of the k-th largest token.  A workgroup per row
// does all this in one launch; a few long rows are divided among many workgroups,
// in three.
#include <hip/hip_runtime.h>

#include <cmath>

#include "it_internal.hpp"
#include "it_rows.hpp"

using namespace itkv;

namespace {
constexpr int kSliceThreads = 512;   // of a slice's workgroup
constexpr int kSliceWaves = kSliceThreads / 64;
constexpr int kThreads = 1024;       // of a row's
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;          // of a row, linear in z
constexpr int kList = 2048;          // tokens listed per row, and gathered in LDS
constexpr int kRowList = 8192;       // room for a row's slices' lists: a slice may hold most of the likely tokens
constexpr int kSliceList = kList - 1;  // of a slice at most: its workgroup's LDS is a quarter of a CU's
constexpr int kFew = 256;            // tokens compared all with all (below)
static_assert(kFew > 64, "narrow() takes more than it for more than a last step's 64");
constexpr int kFineBits = 10, kFine = 1 << kFineBits;
constexpr int kMaxSlices = 32;
constexpr int kGroups = 2 * kSliceWaves;  // group maxima per slice: half waves
constexpr int kMaxVocab = 1 << 18;   // a sum of weights stays below 2^62
constexpr int kRowGroups = kThreads / 2;  // group maxima of such a row, at most
constexpr int kIndexBits = 18;
constexpr double kUnit = 0x1p44;      // weight of the largest token
constexpr double kLeast = 0x1.0000000000001p-45;  // smaller weights round to nothing
constexpr double kBinsPerBit = 44.0;  // of log2 weight, of which 45 weigh at all
static_assert(45 * kBinsPerBit + 2 < kBins, "a bin for every weight");
constexpr uint32_t kDeadKey = 0x007FFFFFu;  // order_key(-inf)

struct RowState {
  uint32_t n_gathered, ticket, pad[30];
  uint32_t n_list[kMaxSlices];              // tokens of each slice that are listed, or more than its room
  uint64_t best[kMaxSlices];               // order of each slice's largest token (the first of equals where the row is greedy), 0: nothing above -inf
  uint32_t group_max[kMaxSlices * kGroups];
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t list[kRowList];                  // by slice; then what the third launch's workgroups gather
};
static_assert(sizeof(RowState) % 256 == 0, "rows of the workspace stay aligned");

__host__ __device__ constexpr int slice_list(int slices) { return kRowList / slices < kSliceList ? kRowList / slices : kSliceList; }

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

// 2^x = 2^n (1 + f h(f)) with n the nearest integer, |f| <= 1/2, and h the
// polynomial through (2^f - 1) / f at the ten Chebyshev nodes of [-1/2, 1/2]: off by
// less than 2^-50 of 2^x, and exactly 1 at x = 0.
constexpr double kExp2[10] = {0x1.62e42fefa39f7p-1,  0x1.ebfbdff82c590p-3,  0x1.c6b08d7044119p-5, 0x1.3b2ab6fba385fp-7, 0x1.5d87fe908f88ap-10,
                              0x1.4309130378460p-13, 0x1.ffcb76789860fp-17, 0x1.62bfe46117445p-20, 0x1.b6571de2f2351p-24, 0x1.e5e9f548e5726p-28};

// An fp64 constant kept in scalar registers: as a literal it would be moved
// into vector registers before each use, twice as much work as the products.
__device__ __forceinline__ double scalar(double x) {
  asm("" : "+s"(x));
  return x;
}
// One kept in vector registers: an instruction reads one scalar operand.
__device__ __forceinline__ double vector(double x) {
  asm("" : "+v"(x));
  return x;
}

// A row's weights, the same in all its threads.  fp64 work bounds them (an fma of
// every token of 256 x 131072 takes 1.4 us of 30), so whole numbers are taken from the
// low word of a sum with 1.5 x 2^52 and exponents are added as integers: 3 us less
// than with fp64's roundings, conversions and ldexp.
struct Weigher {
  float top;      // max z
  float floor;    // tokens below weigh nothing, fail min-p or cannot be among the first k
  double bits;    // log2(e) / T
  double per_bit; // its reciprocal: z for a factor of two
  double least;   // min-p, or the smallest weight that does not round to nothing
  double below;   // z - top of 2^-64; lower ones weigh no more
  double bin_bits, exp2[10], unit, zero, whole;
  __device__ __forceinline__ void constants() {
    // inf - inf is NaN, of which fmax makes 0: tokens at a top of +inf weigh 1.
    below = top < INFINITY ? -64.0 * per_bit : 0.0;
    bin_bits = -kBinsPerBit * bits;
#pragma unroll
    for (int i = 0; i < 10; ++i) exp2[i] = i == 8 ? vector(kExp2[i]) : scalar(kExp2[i]);
    unit = scalar(kUnit);
    zero = vector(0x1p52);
    whole = vector(0x1.8p52);
  }
  // Weight and bin of a token with floor <= z <= top; false: not kept.
  __device__ __forceinline__ bool operator()(float z, uint64_t& w, int& bin) const {
    const double d = fmax(double(z) - double(top), below);
    const double n = fma(d, bits, whole), f = fma(d, bits, whole - n);
    double h = fma(exp2[9], f, exp2[8]);
#pragma unroll
    for (int i = 7; i >= 0; --i) h = fma(h, f, exp2[i]);
    const double m = fma(h, f, 1.0);  // 2^f, above 0.7
    const double e = __hiloint2double(int(uint32_t(__double2hiint(m)) + (uint32_t(__double2loint(n)) << 20)), __double2loint(m));
    // Rounded to a whole number of units by the sum with 2^52.
    w = __builtin_bit_cast(uint64_t, fma(e, unit, zero)) & ((uint64_t(1) << 52) - 1);
    bin = __double2loint(fma(d, bin_bits, whole));  // up to 45 kBinsPerBit for what is kept
    return e >= least;
  }
};

// The tokens of a slice of a row: its share of the 16-byte vectors of the row's
// aligned part, the first slice also the tokens before that part, the last those
// behind it.
template <int DT, int kBlock>
struct Walk {
  static constexpr int es = DT == IT_F32 ? 4 : 2, V = 16 / es;
  using In = RowVec<DT, V>;
  const char* row;
  const typename In::raw* v;
  int vocab, head, done, lo, hi;
  bool first, last;
  typename In::raw next;
  __device__ __forceinline__ Walk(const char* row_, int vocab_, int slice, int slices) : row(row_), vocab(vocab_) {
    head = min(vocab, int((16 - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / es);
    const int vecs = (vocab - head) / V, per = (vecs + slices - 1) / slices;
    done = head + vecs * V;
    lo = min(vecs, slice * per);
    hi = min(vecs, lo + per);
    first = slice == 0;
    last = slice == slices - 1;
    v = reinterpret_cast<const typename In::raw*>(row + head * es);
  }
  // Loads what each() begins with, in the shadow of what a kernel does before it.
  __device__ __forceinline__ void start() {
    if (lo + int(threadIdx.x) < hi) next = v[lo + int(threadIdx.x)];
  }
  template <class F>
  __device__ __forceinline__ void vector(const typename In::raw& w, int x, F&& f) const {
    float z[V];
    In::widen(w, z);
#pragma unroll
    for (int e = 0; e < V; ++e) f(head + x * V + e, z[e]);
  }
  template <class F>
  __device__ __forceinline__ void ends(F&& f) const {
    const int tid = int(threadIdx.x);
    if (first && tid < head) f(tid, load_element(row, tid, DT));
    if (last && tid < vocab - done) f(done + tid, load_element(row, done + tid, DT));
  }
  // f(index, z), once after start(): one vector is loaded while one is worked on.
  // (Batches of vectors in flight read no faster, 16 waves a CU keep enough; and
  // unrolled over them the weighing is 16 to 64 times its code, which small calls
  // wait for.)
  template <class F>
  __device__ __forceinline__ void each(F&& f) {
#pragma unroll 1
    for (int x = lo + int(threadIdx.x); x < hi; x += kBlock) {
      const typename In::raw w = next;
      if (x + kBlock < hi) next = v[x + kBlock];
      vector(w, x, f);
    }
    ends(f);
  }
  // The same of those threads' tokens alone that a thread has `wanted`: where
  // few have, their vectors are shared out among all.  columns: LDS, kBlock
  // places; n: an LDS word.
  template <class F>
  __device__ __forceinline__ void each_wanted(bool wanted, uint32_t* columns, uint32_t* n, F&& f) {
    if (threadIdx.x == 0) *n = 0u;
    __syncthreads();
    if (wanted) columns[atomicAdd(n, 1u)] = threadIdx.x;
    __syncthreads();
    const uint32_t few = *n;
    if (few > kBlock / 2) {
      start();
      each(f);
      return;
    }
    const uint32_t total = few * uint32_t((hi - lo + kBlock - 1) / kBlock);
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < total; i += kBlock) {
      const uint32_t turn = i / few;
      const int x = lo + int(turn * kBlock + columns[i - turn * few]);
      if (x < hi) vector(v[x], x, f);
    }
    ends(f);
  }
};

// x of one lane, the same for all.
__device__ __forceinline__ uint64_t lane64(uint64_t x, int lane) {
  return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(x >> 32), lane))) << 32 | uint32_t(__builtin_amdgcn_readlane(int(x), lane));
}
// The 64-bit x of the lane that a DPP pattern names; 0 for lanes it leaves out.
template <int CTRL, int ROWS = 0xF, int BANKS = 0xF, bool kBound = true>
__device__ __forceinline__ uint64_t dpp64(uint64_t x) {
  const int hi = __builtin_amdgcn_update_dpp(0, int(x >> 32), CTRL, ROWS, BANKS, kBound);
  return uint64_t(uint32_t(hi)) << 32 | uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, ROWS, BANKS, kBound));
}
// The largest of the wave's, in every lane.
__device__ __forceinline__ uint64_t wave_max64(uint64_t x) {
  x = max(x, dpp64<kDppQuadXor1>(x));
  x = max(x, dpp64<kDppQuadXor2>(x));
  x = max(x, dpp64<kDppHalfMirror>(x));
  x = max(x, dpp64<kDppRowRor8>(x));
  return max(max(lane64(x, 0), lane64(x, 16)), max(lane64(x, 32), lane64(x, 48)));
}
// The largest of groups of n lanes, n a power of two up to 32, in every lane of each.
__device__ __forceinline__ uint32_t group_max32(uint32_t x, int n) {
  if (n >= 2) x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppQuadXor1, 0xF, 0xF, true)));
  if (n >= 4) x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppQuadXor2, 0xF, 0xF, true)));
  if (n >= 8) x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppHalfMirror, 0xF, 0xF, true)));
  if (n >= 16) x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), kDppRowRor8, 0xF, 0xF, true)));
  if (n >= 32) x = max(x, uint32_t(__shfl_xor(int(x), 16)));
  return x;
}
// x summed over the lanes up to and with each.
__device__ __forceinline__ uint64_t wave_inclusive_sum64(uint64_t x) {
  uint64_t v = x + dpp64<0x111>(x);          // row_shr:1
  v += dpp64<0x112>(x);                      // row_shr:2
  v += dpp64<0x113>(x);                      // row_shr:3
  v += dpp64<0x114, 0xF, 0xE, false>(v);     // row_shr:4, banks 1-3
  v += dpp64<0x118, 0xF, 0xC, false>(v);     // row_shr:8, banks 2-3
  v += dpp64<0x142, 0xA, 0xF, false>(v);     // row_bcast:15, rows 1, 3
  return v + dpp64<0x143, 0xC, 0xF, false>(v);  // row_bcast:31, rows 2-3
}
// x summed over groups of n lanes, n a power of two up to 16, in every lane of each.
__device__ __forceinline__ uint64_t group_sum64(uint64_t x, uint32_t n) {
  if (n >= 2) x += dpp64<kDppQuadXor1>(x);
  if (n >= 4) x += dpp64<kDppQuadXor2>(x);
  if (n >= 8) x += dpp64<kDppHalfMirror>(x);
  if (n >= 16) x += dpp64<kDppRowRor8>(x);
  return x;
}

// x summed over the wave's lanes up to and with each; returns the sum of all.
__device__ __forceinline__ uint32_t wave_sums(uint32_t& x) {
  x = uint32_t(wave_inclusive_sum(int(x)));
  return uint32_t(__builtin_amdgcn_readlane(int(x), 63));
}

__device__ __forceinline__ float temperature_of(const SampleArgs& a, int row) {
  return a.temperatures ? a.temperatures[row] : a.temperature;
}
// A thread's largest token, and which it is where the row takes the first of the
// order: the index is three more instructions a token, which took one workgroup 2
// us of the 4 for 32000.
template <class W>
__device__ __forceinline__ void find_top(W& walk, bool greedy, float& top, int& at) {
  top = -INFINITY;
  at = 0;
  if (greedy) {  // uniform
    walk.each([&](int i, float z) {
      if (z > top || (z == top && i < at)) top = z, at = i;
    });
  } else {
    walk.each([&](int, float z) { top = fmaxf(top, z); });
  }
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_maxima(SampleArgs a) {
  __shared__ uint64_t best_of[kSliceWaves];
  const int slice = int(blockIdx.x), lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6);
  RowState& rs = a.rows[blockIdx.y];
  if (slice == 0 && threadIdx.x == 0)  // what the second launch adds to
    rs.n_gathered = rs.ticket = 0u;
  for (int b = slice * kSliceThreads + int(threadIdx.x); b < kBins; b += a.slices * kSliceThreads) rs.count[b] = 0u, rs.mass[b] = 0u;
  float top;
  int at;
  Walk<DT, kSliceThreads> walk(a.logits + int64_t(blockIdx.y) * a.row_bytes, a.vocab, slice, a.slices);
  walk.start();
  find_top(walk, !(temperature_of(a, int(blockIdx.y)) > 0.0f), top, at);
  uint64_t best = top > -INFINITY ? order_of(top, at) : 0u;
  const uint32_t group = group_max32(order_key(top), 32);
  if ((lane & 31) == 0) rs.group_max[slice * kGroups + wave * 2 + (lane >> 5)] = group;
  best = wave_max64(best);
  if (lane == 0) best_of[wave] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSliceWaves; ++i) best = best_of[i] > best ? best_of[i] : best;
    rs.best[slice] = best;
  }
}

// A row's settings, as all its workgroups derive them from the first launch's
// maxima; false where there is nothing to weigh: an empty row, or one that takes
// the first of the order (best is its place).
struct Settings {
  Weigher weigh;
  uint64_t best;
  int top_k, groups;
  bool listed;  // few tokens can be kept: they are listed
  static constexpr int kLoads = kMaxSlices * kGroups / 64;
  uint32_t group[kLoads];
  __device__ __forceinline__ bool plain() const { return !listed && top_k <= 0; }  // uniform
  // The group maxima, 64 to a register, before it is known whether they count.
  __device__ __forceinline__ void load_groups(const SampleArgs& a, const uint32_t* maxima, int n) {
    const int lane = int(threadIdx.x & 63);
    groups = n;
    if (!a.top_ks && a.top_k <= 0) return;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = j * 64 + lane;
      group[j] = i < groups ? maxima[i] : 0u;
    }
  }
  // first: the place of the row's largest token, 0 where nothing is above -inf.
  __device__ __forceinline__ bool derive(const SampleArgs& a, int row, uint64_t first) {
    const float temp = temperature_of(a, row);
    const float min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    best = lane64(first, 0);
    if (best == 0u || !(temp > 0.0f)) return false;  // uniform
    weigh.top = order_value(best);
    weigh.bits = 1.4426950408889634 / double(temp);
    weigh.per_bit = 0.6931471805599453 * double(temp);
    const double share = min_p > 0.0f ? fmin(double(min_p), 1.0) : 0.0;  // NaN: off
    weigh.least = fmax(share, kLeast);
    // Below floor a weight is below `least`: z - top < T ln(least), widened by
    // fp32's rounding.
    weigh.floor = weigh.top;
    if (weigh.top < INFINITY) {
      const double low = double(weigh.top) + (share > kLeast ? log2(share) : -45.0) * weigh.per_bit;
      weigh.floor = float(low - fabs(low) * 0x1p-20);
    }
    // Whatever the floor, a token at -inf is never kept.
    weigh.floor = fmaxf(weigh.floor, -3.402823466e38f);
    listed = share > 0.0 || (top_k > 0 && top_k <= groups);
    return true;
  }
  // The floor raised to the first sixteen bits of the top_k-th largest group
  // maximum: at least top_k tokens have keys that large.
  __device__ __forceinline__ void raise_floor() {
    if (top_k <= 0 || top_k > groups) return;
    const uint32_t key = groups <= 128 ? search<2>() : search<kLoads>();
    if (key > kDeadKey) weigh.floor = fmaxf(weigh.floor, key_value(key));
  }
  template <int N>
  __device__ __forceinline__ uint32_t search() const {
    uint32_t key = 0u;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t with = key | 1u << bit;
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) n += __popcll(__ballot(group[j] >= with));
      if (n >= top_k) key = with;
    }
    return key;
  }
  // What a row without anything to weigh answers.
  __device__ __forceinline__ void trivial(const SampleArgs& a, int row) const {
    a.tokens[row] = best ? order_index(best) : -1;
    if (a.probs) a.probs[row] = best ? 1.0f : 0.0f;
  }
};

// Adds a token to a workgroup's bins, and to its list of `room` places where
// few tokens can be kept.
__device__ __forceinline__ void weigh_token(const Settings& set, float z, int index, uint64_t* mass, uint32_t* count, uint64_t* list,
                                            uint32_t* n, uint32_t room) {
  if (!(z >= set.weigh.floor)) return;
  uint64_t w;
  int b;
  if (!set.weigh(z, w, b)) return;
  atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), (unsigned long long)(w));
  if (set.top_k > 0) atomicAdd(&count[b], 1u);  // only top-k asks for counts
  if (set.listed) {
    const uint32_t at = atomicAdd(n, 1u);
    if (at < room) list[at] = order_of(z, index);
  }
}

// The same where no list or count is asked for: one branch a token (256 x 131072 with
// top-p 76.2 -> 72.4 us, 1 x 32000 whole 15.9 -> 14.5).
__device__ __forceinline__ void weigh_plain(const Settings& set, float z, uint64_t* mass) {
  uint64_t w;
  int b;
  const int kept = int(set.weigh(z, w, b)) & int(z >= set.weigh.floor);
  if (kept) atomicAdd(reinterpret_cast<unsigned long long*>(&mass[b]), (unsigned long long)(w));
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads, 8) void sample_weigh(SampleArgs a) {
  __shared__ uint64_t mass[kBins], list[kSliceList];
  __shared__ uint32_t count[kBins], n;
  const int t = int(threadIdx.x), slice = int(blockIdx.x), row = int(blockIdx.y);
  RowState& rs = a.rows[row];
  Walk<DT, kSliceThreads> walk(a.logits + int64_t(row) * a.row_bytes, a.vocab, slice, a.slices);
  walk.start();
  Settings set;
  set.load_groups(a, rs.group_max, a.slices * kGroups);
  if (!set.derive(a, row, wave_max64((t & 63) < a.slices ? rs.best[t & 63] : 0u))) return;
  set.raise_floor();
  set.weigh.constants();
  for (int b = t; b < kBins; b += kSliceThreads) count[b] = 0u, mass[b] = 0u;
  if (t == 0) n = 0u;
  __syncthreads();
  const uint32_t room = slice_list(a.slices);
  if (set.plain()) walk.each([&](int, float z) { weigh_plain(set, z, mass); });
  else walk.each([&](int i, float z) { weigh_token(set, z, i, mass, count, list, &n, room); });
  __syncthreads();
  if (set.listed) {  // each slice in its own part of the row's list
    if (t == 0) rs.n_list[slice] = n;
    if (n <= room)
      for (uint32_t i = t; i < n; i += kSliceThreads) rs.list[slice * room + i] = list[i];
  }
  for (int b = t; b < kBins; b += kSliceThreads) {
    if (mass[b] == 0u) continue;
    atomicAdd(reinterpret_cast<unsigned long long*>(&rs.mass[b]), (unsigned long long)(mass[b]));
    if (set.top_k > 0) atomicAdd(&rs.count[b], count[b]);
  }
}

struct Shared {
  uint64_t mass[kBins];   // the row's bins
  uint64_t cand[kList];   // the tokens gathered to answer from
  struct Weighed {
    uint64_t order, weight;
  };
  union {
    uint64_t fine[kFine];          // narrow(): bins inside a bin
    Weighed weighed[kFew];         // answer_from()
  };
  uint32_t count[kBins];
  uint32_t fine_count[kFine];
  Weighed last[64];
  uint64_t wave_mass[kWaves];
  uint32_t wave_count[kWaves];
  uint32_t n, base;
  uint64_t kept[2];
  struct Found {
    uint64_t before_mass, mass;
    uint32_t before_count, count, bin;
  } found[5];
  uint64_t weight, mass_to;
  int token;
};

// Sums over the threads before this one, and over all.
struct Scan {
  uint64_t mass, total_mass;
  uint32_t count, total_count;
};
__device__ __forceinline__ Scan block_scan(Shared& s, uint32_t count, uint64_t mass) {
  const int lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6);
  const uint32_t c = uint32_t(wave_inclusive_sum(int(count)));
  const uint64_t m = wave_inclusive_sum64(mass);
  __syncthreads();  // the sums of the call before are read
  if (lane == 63) s.wave_count[wave] = c, s.wave_mass[wave] = m;
  __syncthreads();
  static_assert(kWaves == 16, "a wave's sums in each lane of a DPP row");
  const uint32_t wave_c = s.wave_count[lane & 15];
  const uint64_t wave_m = s.wave_mass[lane & 15], to_m = wave_inclusive_sum64(lane < 16 ? wave_m : 0u);
  const uint32_t to_c = uint32_t(wave_inclusive_sum(int(lane < 16 ? wave_c : 0u)));
  const uint64_t before_m = lane64(to_m, wave) - lane64(wave_m, wave);
  const uint32_t before_c = uint32_t(__builtin_amdgcn_readlane(int(to_c), wave) - __builtin_amdgcn_readlane(int(wave_c), wave));
  return {before_m + m - mass, lane64(to_m, 15), before_c + c - count, uint32_t(__builtin_amdgcn_readlane(int(to_c), 15))};
}

// What is before a thread's N consecutive bins of LDS, which stay there.
template <int N>
struct Bins {
  uint64_t before_mass, total_mass;
  uint32_t before_count, total_count;
  __device__ __forceinline__ Bins(Shared& s, const uint32_t* c, const uint64_t* m, uint32_t base_count, uint64_t base_mass) {
    uint32_t cs = 0u;
    uint64_t ms = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) cs += c[N * threadIdx.x + i], ms += m[N * threadIdx.x + i];
    const Scan scan = block_scan(s, cs, ms);
    before_count = base_count + scan.count;
    before_mass = base_mass + scan.mass;
    total_count = base_count + scan.total_count;
    total_mass = base_mass + scan.total_mass;
  }
  // The one bin in which the cumulative count (or mass) reaches `goal`, 1 <=
  // goal <= the total, into `f` (a barrier later).
  __device__ __forceinline__ void find(const uint32_t* c, const uint64_t* m, Shared::Found& f, bool by_count, uint64_t goal) const {
    uint32_t cs = before_count;
    uint64_t ms = before_mass;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t ci = c[N * threadIdx.x + i];
      const uint64_t mi = m[N * threadIdx.x + i];
      const uint64_t before = by_count ? cs : ms, after = before + (by_count ? uint64_t(ci) : mi);
      if (before < goal && goal <= after) f = {ms, mi, cs, ci, uint32_t(N * threadIdx.x + i)};
      cs += ci;
      ms += mi;
    }
  }
};

template <int DT>
struct Row {
  const char* data;
  int vocab;
  Weigher weigh;
  // f(order, z) for the row's tokens with lo <= z <= hi.
  template <class F>
  __device__ __forceinline__ void each(float lo, float hi, F&& f) const {
    Walk<DT, kThreads> walk(data, vocab, 0, 1);
    walk.start();
    walk.each([&](int i, float z) {
      if (z >= lo && z <= hi) f(order_of(z, i), z);
    });
  }
  // The z of bins first .. last, widened by what rounding can move an edge.
  __device__ __forceinline__ void span(int first, int last, float& lo, float& hi) const {
    lo = weigh.floor;
    hi = INFINITY;
    if (weigh.top < INFINITY && weigh.per_bit < double(INFINITY)) {
      const double edge = weigh.per_bit / kBinsPerBit, top = double(weigh.top);
      const double begin = top - (double(first) - 0.5) * edge, end = top - (double(last) + 0.5) * edge;
      hi = float(begin + (fabs(begin) + edge) * 0x1p-20);
      lo = fmaxf(lo, float(end - (fabs(end) + edge) * 0x1p-20));
    }
  }
};

// Where top-k ends, where top-p ends (each leaves the mass kept), the draw: the
// goal of each as a function of the mass kept so far, which none decreases with.
struct Questions {
  uint64_t top_k;  // 0: off
  float top_p, u;
  __device__ __forceinline__ bool cuts() const { return top_p < 1.0f; }  // NaN: off
  __device__ __forceinline__ uint64_t cut(uint64_t kept) const {
    // before < top_p kept  <=>  before < ceil(top_p kept), before being whole.
    const double part = top_p > 0.0f ? ceil(double(top_p) * double(kept)) : 0.0;
    const uint64_t goal = part < 1.0 ? 1u : uint64_t(part);
    return goal < kept ? goal : kept;
  }
  __device__ __forceinline__ uint64_t draw(uint64_t kept) const {
    const uint64_t goal = u > 0.0f ? uint64_t(fmin(double(u), 1.0) * double(kept)) : 0u;  // kept <= 2^62
    return (goal < kept ? goal : kept - 1) + 1;
  }
};

// All answers from the n <= kFew tokens in s.cand (a barrier before), which are all
// that may be kept.
// Each one's place is found by comparing it with all others, a power of two of
// threads sharing them: no step waits for the one before, but the work grows with
// n^2.  1 x 32000 with top-k 100, which lists 129 to 256 tokens, takes 13.0 us, and
// 20.0 by bins; with 120, 257 to 512 tokens, 27.4 all with all and 21.6 by bins.
template <int DT>
__device__ __forceinline__ void answer_from(Shared& s, const Row<DT>& row, const Questions& ask, uint32_t n, const SampleArgs& a,
                                            int out) {
  const int t = int(threadIdx.x);
  int log2_parts = 0;
  while (log2_parts < 4 && uint32_t(kThreads >> (log2_parts + 1)) >= n) ++log2_parts;
  const uint32_t parts = 1u << log2_parts;
  Shared::Weighed* const all = s.weighed;
  uint64_t own = 0u, w = 0u;
  int bin = 0;
  if (t < int(n)) {
    own = s.cand[t];
    row.weigh(order_value(own), w, bin);
    all[t] = {own, w};
  }
  __syncthreads();
  const uint32_t i = uint32_t(t) >> log2_parts, part = uint32_t(t) & (parts - 1);
  own = i < n ? all[i].order : ~0ull;
  uint32_t before_count = 0u;
  uint64_t before_mass = 0u, kept = 0u;
#pragma unroll 4
  for (uint32_t j = part; j < n; j += parts) {
    const Shared::Weighed x = all[j];
    kept += x.weight;
    if (x.order > own) before_count += 1u, before_mass += x.weight;
  }
  kept = group_sum64(kept, parts);
  before_mass = group_sum64(before_mass, parts);
  before_count = uint32_t(group_sum64(before_count, parts));
  w = i < n ? all[i].weight : 0u;
  const bool one = i < n && part == 0;
  // f() for the token at which the count, or the mass, reaches the goal.
  const auto at = [&](bool by_count, uint64_t goal, auto&& f) {
    const uint64_t before = by_count ? uint64_t(before_count) : before_mass, after = before + (by_count ? 1u : w);
    if (one && before < goal && goal <= after) f();
  };
  if (ask.top_k > 0 && ask.top_k < n) {
    at(true, ask.top_k, [&] { s.kept[0] = before_mass + w; });
    __syncthreads();
    kept = s.kept[0];
  }
  if (ask.cuts()) {
    at(false, ask.cut(kept), [&] { s.kept[1] = before_mass + w; });
    __syncthreads();
    kept = s.kept[1];
  }
  at(false, ask.draw(kept), [&] {
    a.tokens[out] = order_index(own);
    if (a.probs) a.probs[out] = float(double(w) / double(kept));
  });
}

// One question over any number of tokens (many equal logits, a flat row): bins
// inside the bin f, a power of two of orders each, until 64 tokens are left.
// gathered: s.cand holds that many tokens, all of the bin's among them; past kList
// they are read from the row, again each time until they fit.  The answer is
// s.token, its weight, and the mass up to and with it in s.mass_to.
template <int DT>
__device__ __forceinline__ void narrow(Shared& s, const Row<DT>& row, const Shared::Found& f, bool by_count, uint64_t goal,
                                       uint32_t gathered) {
  const int t = int(threadIdx.x), bin = int(f.bin);
  uint32_t n, bc = f.before_count;
  uint64_t bm = f.before_mass;
  float zlo, zhi;
  row.span(bin, bin, zlo, zhi);
  uint64_t lo = order_of(zlo, kMaxVocab - 1), hi = order_of(fminf(zhi, row.weigh.top), 0);
  bool held = gathered <= kList;  // in s.cand
  uint32_t cands = gathered;
  // g(order, weight) for the bin's tokens with lo <= order <= hi.
  const auto each_in = [&](auto&& g) {
    const auto member = [&](uint64_t o, float z) {
      uint64_t w;
      int b;
      if (o >= lo && o <= hi && row.weigh(z, w, b) && b == bin) g(o, w);
    };
    if (held) {
      for (uint32_t i = t; i < cands; i += kThreads) member(s.cand[i], order_value(s.cand[i]));
    } else {
      row.each(order_value(lo), order_value(hi), member);
    }
  };
  // Their number; the first 64 of them in s.last.  s.n is 0 before, as it is when
  // narrow() begins, and at the end of each turn below.
  const auto collect = [&] {
    each_in([&](uint64_t o, uint64_t w) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < 64) s.last[at] = {o, w};
    });
    __syncthreads();
    return s.n;
  };
  n = gathered <= kFew ? collect() : kFew;
  // Nine bits of hi - lo < 2^50 a turn or more; orders are unique.
  for (int turn = 0; n > 64 && turn < 6; ++turn) {
    const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - kFineBits);
    __syncthreads();
    for (int b = t; b < kFine; b += kThreads) s.fine_count[b] = 0u, s.fine[b] = 0u;
    __syncthreads();
    each_in([&](uint64_t o, uint64_t w) {
      const uint32_t x = uint32_t((hi - o) >> shift);
      atomicAdd(&s.fine_count[x], 1u);
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.fine[x]), (unsigned long long)(w));
    });
    __syncthreads();
    const Bins<kFine / kThreads> fine(s, s.fine_count, s.fine, bc, bm);
    fine.find(s.fine_count, s.fine, s.found[4], by_count, goal);
    if (t == 0) s.n = 0u;
    __syncthreads();
    n = s.found[4].count;
    bc = s.found[4].before_count;
    bm = s.found[4].before_mass;
    hi -= uint64_t(s.found[4].bin) << shift;
    const uint64_t width = uint64_t(1) << shift;
    lo = hi >= width && hi - width + 1 > lo ? hi - width + 1 : lo;
    if (n <= 64) {  // uniform
      n = collect();
      break;
    }
    if (!held && n <= kList) {
      each_in([&](uint64_t o, uint64_t) {
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < kList) s.cand[at] = o;
      });
      held = true;
      cands = n;
    }
  }
  // Sixteen threads a token sum the mass of those up to it.
  n = min(n, 64u);
  const uint32_t i = uint32_t(t) >> 4;
  const Shared::Weighed own = i < n ? s.last[i] : Shared::Weighed{~0ull, 0u};
  uint32_t ci = 0u;
  uint64_t mi = 0u;
#pragma unroll
  for (uint32_t j = uint32_t(t) & 15u; j < 64u; j += 16u) {
    if (j >= n) continue;
    const Shared::Weighed x = s.last[j];
    if (x.order >= own.order) ci += 1u, mi += x.weight;
  }
  ci = uint32_t(group_sum64(ci, 16));
  mi = group_sum64(mi, 16);
  const uint64_t after = by_count ? uint64_t(bc + ci) : bm + mi, before = by_count ? after - 1 : after - own.weight;
  if (i < n && (t & 15) == 0 && before < goal && goal <= after) {
    s.token = order_index(own.order);
    s.weight = own.weight;
    s.mass_to = bm + mi;
  }
  __syncthreads();
}

// The z of the tokens to answer from, once a row's bins are in s.count and s.mass.
template <int DT>
struct Plan {
  Bins<kBins / kThreads> bins;
  bool by_k;
  float lo[3], hi[3], lowest;
  // The bins that the answers lie in: a question's goal is known within the mass
  // of the bin that the one before it ends in.
  __device__ __forceinline__ Plan(Shared& s, const Row<DT>& row, const Questions& ask) : bins(s, s.count, s.mass, 0u, 0u) {
    uint64_t low = bins.total_mass, high = low;  // bounds of the mass kept
    by_k = ask.top_k > 0 && ask.top_k < bins.total_count;  // counts are there with top-k alone
    uint32_t k_bin = 0u, p_first = 0u, p_last = 0u;
    if (by_k) {
      bins.find(s.count, s.mass, s.found[0], true, ask.top_k);
      __syncthreads();
      k_bin = s.found[0].bin;
      low = s.found[0].before_mass + 1;
      high = s.found[0].before_mass + s.found[0].mass;
    }
    if (ask.cuts()) {
      bins.find(s.count, s.mass, s.found[1], false, ask.cut(low));
      bins.find(s.count, s.mass, s.found[2], false, ask.cut(high));
      __syncthreads();
      p_first = s.found[1].bin;
      p_last = s.found[2].bin;
      low = ask.cut(low);
      const uint64_t to = s.found[2].before_mass + s.found[2].mass;
      high = to < high ? to : high;
    }
    // All of this is fp64 and 64-bit work in all waves of the workgroup: what nothing
    // asks for is left out.
    bins.find(s.count, s.mass, s.found[3], false, ask.draw(low));
    if (low != high) bins.find(s.count, s.mass, s.found[4], false, ask.draw(high));
    if (threadIdx.x == 0) s.n = 0u;
    __syncthreads();
    row.span(int(s.found[3].bin), int(s.found[low != high ? 4 : 3].bin), lo[0], hi[0]);
    lo[1] = lo[2] = lowest = lo[0];
    hi[1] = hi[2] = hi[0];
    if (ask.cuts()) row.span(int(p_first), int(p_last), lo[1], hi[1]);
    if (by_k) row.span(int(k_bin), int(k_bin), lo[2], hi[2]);
    lowest = fminf(fminf(lowest, lo[1]), lo[2]);
  }
  // A token of the row into s.cand, if it is one of them; their number in s.n.
  template <class F>
  __device__ __forceinline__ void gather(Shared& s, float z, F&& order) const {
    // Two instructions a range and one branch: with compares and branches a row of
    // 32000 whose draw lies among its many took 24.4 us, with these 21.3.
    const auto within = [&](int i) { return int(__builtin_amdgcn_fmed3f(z, lo[i], hi[i]) == z); };
    if (!(within(0) | within(1) | within(2))) return;
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kList) s.cand[at] = order();
  }
  // The answers, from the n tokens gathered (from the row where they are too many).
  __device__ __forceinline__ void answer(Shared& s, const Row<DT>& row, const Questions& ask, uint32_t n, const SampleArgs& a,
                                         int out) const {
    uint64_t kept = bins.total_mass;
    __syncthreads();
    for (int question = by_k ? 0 : 1; question < 3; ++question) {
      if (question == 1 && !ask.cuts()) continue;
      const uint64_t goal = question == 0 ? ask.top_k : question == 1 ? ask.cut(kept) : ask.draw(kept);
      const bool known = question == 2 && !by_k && !ask.cuts();  // the plan's first answer
      if (!known) bins.find(s.count, s.mass, s.found[question], question == 0, goal);
      if (threadIdx.x == 0) s.n = 0u;
      __syncthreads();
      narrow(s, row, s.found[known ? 3 : question], question == 0, goal, n);
      if (question < 2) kept = s.mass_to;
    }
    if (threadIdx.x == 0) {
      a.tokens[out] = s.token;
      if (a.probs) a.probs[out] = float(double(s.weight) / double(kept));
    }
  }
};
__device__ __forceinline__ Questions questions(const SampleArgs& a, const Settings& set, int row) {
  return {set.top_k > 0 ? uint64_t(set.top_k) : 0u, a.top_ps ? a.top_ps[row] : a.top_p, a.u[row]};
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_draw(SampleArgs a) {
  __shared__ Shared s;
  const int t = int(threadIdx.x), part = int(blockIdx.x), parts = int(gridDim.x), row = int(blockIdx.y);
  RowState& rs = a.rows[row];
  // Read before they are known to be needed: one wait for all of them.
  uint32_t counts[kBins / kThreads];
  uint64_t masses[kBins / kThreads];
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) counts[i] = rs.count[i * kThreads + t], masses[i] = rs.mass[i * kThreads + t];
  const uint32_t listed_here = rs.n_list[t & (kMaxSlices - 1)];  // lane i: of slice i (not written where nothing is listed)
  Settings set;
  set.groups = a.slices * kGroups;
  if (!set.derive(a, row, wave_max64((t & 63) < a.slices ? rs.best[t & 63] : 0u))) {  // uniform
    if (t == 0 && part == 0) set.trivial(a, row);
    return;
  }
  const Questions ask = questions(a, set, row);
  set.weigh.constants();
  Row<DT> r{a.logits + int64_t(row) * a.row_bytes, a.vocab, set.weigh};
  // Every token that may be kept is listed, unless there are too many.
  const uint32_t room = slice_list(a.slices);
  uint32_t n_list = (t & 63) < a.slices && set.listed ? listed_here : 0u, list_at = n_list;
  const bool fits = !__any(n_list > room);
  const uint32_t n_listed = wave_sums(list_at);
  const bool from_list = set.listed && fits && n_listed <= kList;
  if (from_list && part) return;
  // f(order, place) for them.
  const auto each_listed = [&](auto&& f) {
    for (int i = t >> 6; i < a.slices; i += kWaves) {
      const uint32_t n = uint32_t(__shfl(int(n_list), i)), at = uint32_t(__shfl(int(list_at), i)) - n;
      for (uint32_t j = t & 63; j < n; j += 64) f(rs.list[i * room + j], at + j);
    }
  };
  if (from_list && n_listed <= kFew) {
    each_listed([&](uint64_t o, uint32_t at) { s.cand[at] = o; });
    __syncthreads();
    answer_from(s, r, ask, n_listed, a, row);
    return;
  }
  set.load_groups(a, rs.group_max, a.slices * kGroups);
  set.raise_floor();
  r.weigh.floor = set.weigh.floor;
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) s.count[i * kThreads + t] = counts[i], s.mass[i * kThreads + t] = masses[i];
  __syncthreads();
  const Plan<DT> plan(s, r, ask);
  // A row's workgroups have all come here alike; each gathers its part.
  if (from_list) {
    each_listed([&](uint64_t o, uint32_t) { plan.gather(s, order_value(o), [&] { return o; }); });
  } else {
    Walk<DT, kThreads> walk(r.data, a.vocab, part, parts);
    walk.start();
    walk.each([&](int i, float z) { plan.gather(s, z, [&] { return order_of(z, i); }); });
  }
  __syncthreads();
  uint32_t n = s.n;
  if (parts > 1 && !from_list) {
    // The row's last workgroup answers, from what all of them gathered.  What
    // passes between them goes through device-scope atomics, which meet behind the
    // XCDs' caches: each wave waits for its own to be acknowledged before the
    // ticket is taken, and the last one's loads follow its ticket.  A device-scope
    // fence would do the same by writing back and dropping the XCD's L2, for 20 to
    // 35 us in each workgroup of a large call.
    if (t == 0) s.base = atomicAdd(&rs.n_gathered, n <= kList ? n : uint32_t(kList + 1));
    __syncthreads();
    if (n <= kList && s.base + n <= kList)
      for (uint32_t i = t; i < n; i += kThreads)
        __hip_atomic_store(&rs.list[s.base + i], s.cand[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) s.base = atomicAdd(&rs.ticket, 1u);
    __syncthreads();
    if (s.base != uint32_t(parts - 1)) return;  // uniform
    n = __hip_atomic_load(&rs.n_gathered, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (n <= kList)
      for (uint32_t i = t; i < n; i += kThreads)
        s.cand[i] = __hip_atomic_load(&rs.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  plan.answer(s, r, ask, n, a, row);
}

// All three launches' work by one workgroup per row, whose bins and list stay in
// its LDS: for rows that one CU weighs in the time that two more launches would
// take, and for batches that fill the device so (see row_per_workgroup).
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_row(SampleArgs a) {
  __shared__ Shared s;
  __shared__ uint32_t maxima[kRowGroups];
  const int t = int(threadIdx.x), lane = t & 63, row = int(blockIdx.x);
  const char* const data = a.logits + int64_t(row) * a.row_bytes;
  float top;
  int at;
  Walk<DT, kThreads> walk(data, a.vocab, 0, 1);
  walk.start();
  for (int b = t; b < kBins; b += kThreads) s.count[b] = 0u, s.mass[b] = 0u;
  find_top(walk, !(temperature_of(a, row) > 0.0f), top, at);
  // Groups of eight lanes; of two where threads have no tokens: top-k 50 of 1000
  // would find 31 groups, and take 18.1 us for its long list instead of 9.3
  // (4096: 7.7 with groups of eight, 9.1 of two, a longer floor search).
  const int log2_lanes = walk.hi - walk.lo >= kThreads ? 3 : 1;
  const uint32_t group = group_max32(order_key(top), 1 << log2_lanes);
  if ((lane & ((1 << log2_lanes) - 1)) == 0) maxima[t >> log2_lanes] = group;
  const uint64_t best = wave_max64(top > -INFINITY ? order_of(top, at) : 0u);
  if (lane == 0) s.wave_mass[t >> 6] = best;
  if (t == 0) s.n = 0u;
  __syncthreads();
  Settings set;
  set.load_groups(a, maxima, kThreads >> log2_lanes);
  if (!set.derive(a, row, wave_max64(lane < kWaves ? s.wave_mass[lane] : 0u))) {  // uniform
    if (t == 0) set.trivial(a, row);
    return;
  }
  set.raise_floor();
  set.weigh.constants();
  const Questions ask = questions(a, set, row);
  const Row<DT> r{data, a.vocab, set.weigh};
  // A thread whose largest token is below the floor has none to weigh: with top-k
  // 50 of 256 x 131072 the call takes 32 us instead of 41.
  if (set.plain()) {
    walk.start();
    walk.each([&](int, float z) { weigh_plain(set, z, s.mass); });
  } else {
    walk.each_wanted(top >= set.weigh.floor, s.fine_count, &s.base,
                     [&](int i, float z) { weigh_token(set, z, i, s.mass, s.count, s.cand, &s.n, kList); });
  }
  __syncthreads();
  const uint32_t n_listed = s.n;
  if (set.listed && n_listed <= kFew) {
    answer_from(s, r, ask, n_listed, a, row);
    return;
  }
  __syncthreads();
  const Plan<DT> plan(s, r, ask);
  uint32_t n = n_listed;  // a list holds all that can be asked for
  if (!set.listed || n_listed > kList) {
    walk.each_wanted(top >= plan.lowest, s.fine_count, &s.base,
                     [&](int i, float z) { plan.gather(s, z, [&] { return order_of(z, i); }); });
    __syncthreads();
    n = s.n;
  }
  plan.answer(s, r, ask, n, a, row);
}

// One launch of a workgroup per row, or three of many per row.  us, f32, T 1 whole / T
// 0.8, top-k 50 and top-p 0.95 / top-p 0.9, one launch against three: 1 x 4096 8.3 /
// 7.8 / 10.8 against 13.7 / 18.4 / 15.9; 1 x 32768 14.6 / 9.1 / 17.1 against 16.0 /
// 14.4 / 18.2; 1 x 50000 18.3 / 9.3 / 21.7 against 16.1 / 14.3 / 18.3; 64 x 65536 26.4
// / 10.5 / 26.6 against 25.1 / 17.3 / 27.4; 128 x 65536 27.5 / 11.2 / 27.4 against 34.4
// / 24.0 / 36.6; 128 x 100000 41.1 / 17.9 / 44.1 against 42.8 / 27.8 / 45.1; 256 x
// 131072, a row for each CU, 66.1 / 31.3 / 73.5 against 81.3 / 53.1 / 81.9.
// The limits were set for a slower sample_row and are lower than these figures would
// put them: a whole row and top-p cross at about 800 to 1000 times the rows, and with
// top-k one launch is the faster of the two at every size here, so that 128 x 100000
// takes up to 10 us, 64 x 65536 and 1 x 50000 5 to 7 longer than they might.
bool row_per_workgroup(int32_t rows, int32_t vocab) { return vocab <= 32768 || vocab <= 512 * int64_t(rows); }

// Slices of a row in the first two launches: of 2048 tokens or more; two workgroups
// on each of 256 CUs, each of which adds its bins to the row's; up to four where a row
// would have fewer than eight slices, whose maxima bound top-k up to 128.  us with
// two / three / four workgroups a CU (eight slices a row, twelve, sixteen), 64 x 100003
// bf16: whole 27.7 / 28.3 / 29.5, T 0.8 with top-k 50 and top-p 0.95 18.0 / 21.7 / 24.2,
// top-p 0.9 29.7 / 30.3 / 31.7.  The result does not depend on it, nor on the
// workgroups that gather in the third.
int slice_count(int32_t rows, int32_t vocab) {
  int s = (vocab + 2047) / 2048;
  const int most = 1024 / rows > 0 ? 1024 / rows : 1, least = most < 8 ? most : 8;
  const int fill = 512 / rows > least ? 512 / rows : least;
  s = s < fill ? s : fill;
  return s < kMaxSlices ? s : kMaxSlices;
}
// Workgroups of a row in the third: of 8192 tokens or more, 256 in all (the same
// calls, whole / top-p 0.9: 27.7 / 29.7 us; one per row 30.2 / 32.2, 512 in all 35.7 /
// 39.6).
int part_count(int32_t rows, int32_t vocab) {
  const int p = (vocab + 8191) / 8192, fill = 256 / rows > 0 ? 256 / rows : 1;
  return p < fill ? p : fill;
}

template <int DT>
void launch_sample(const SampleArgs& a, int32_t rows, hipStream_t s) {
  if (row_per_workgroup(rows, a.vocab)) {
    hipLaunchKernelGGL(sample_row<DT>, dim3(unsigned(rows)), dim3(kThreads), 0, s, a);
    return;
  }
  const dim3 grid(unsigned(a.slices), unsigned(rows));
  hipLaunchKernelGGL(sample_maxima<DT>, grid, dim3(kSliceThreads), 0, s, a);
  hipLaunchKernelGGL(sample_weigh<DT>, grid, dim3(kSliceThreads), 0, s, a);
  hipLaunchKernelGGL(sample_draw<DT>, dim3(unsigned(part_count(rows, a.vocab)), unsigned(rows)), dim3(kThreads), 0, s, a);
}
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
}  // namespace

extern "C" size_t it_sample_workspace(int32_t n_rows, int32_t vocab) {
  return n_rows > 0 && vocab > 0 && !row_per_workgroup(n_rows, vocab) ? size_t(n_rows) * sizeof(RowState) : 0;
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
  const size_t need = it_sample_workspace(n_rows, vocab);
  if (need && (!ws || ws_bytes < need || !aligned(ws, 256)))
    return fail(IT_INVALID_INPUT, "%s: workspace of %zu bytes, %zu needed, 256-byte aligned", who, ws ? ws_bytes : size_t(0), need);
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
