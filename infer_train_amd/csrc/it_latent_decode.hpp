// it_latent_decode.hpp -- absorbed latent attention over the paged cache on the
// matrix cores (F16 and BF16 rows of the usual widths).
//
// All heads of a sequence's new tokens are the query rows of one problem: M =
// q_len * n_heads of them read the same cached rows [c | r] (L + R elements),
// whose first L are the values too:
//   S^T = K Q^T    v_mfma_f32_16x16x32, cached tokens are its rows, queries its
//                  columns, so a lane owns one query: its maximum and sum are
//                  in-lane plus two swaps between the wave's quarters;
//   O^T += C^T P^T the probabilities go back into operands straight from the S^T
//                  registers; C^T comes from the same tile in LDS, transposed on
//                  the way out (ds_read_b64_tr_b16), so a cached row is loaded
//                  from memory once and staged once for both products.
// A wave takes 16 queries and all L values: at L = 512 O^T is 128 registers and Q
// 72, two waves a SIMD.  (32 queries a wave halve the LDS reads, but O^T then is
// 256 registers, which the compiler does not keep in place.)  A workgroup has QG
// query groups that share each 32-token tile and KG token groups, joined in LDS at
// the end.
// Tiles come by direct loads into LDS, as many ahead as fit in 144 KB: at L = 512 three
// where there is one token group, one where there are two, none where there are four.
// Work is divided by tiles over all sequences of the call (Division, below); pieces of
// sequences go through the workspace, at most two of a workgroup, and a second kernel
// joins them.
// Bound by HBM up to about 64 queries (2 (2 L + R) M flops for 2 (L + R) bytes a
// token), by LDS reads and products in turn beyond.  With the join, L = 512 in bf16: 32
// sequences of 256 to 8192 tokens, 32 heads, 41 us (151 MB at 3.7 TB/s; a copy reaches
// 6.65); 16 of 8192 to 16384, 128 heads, 100 us (226 MB; 16 us of them the join of 64 MB of
// partial results); one of 1023, 28 heads, 15 us, all latency (launches, lengths, pages,
// tile, join, one after another).  L = 256 in f16: 24 of 100 to 4096, four drafted tokens
// of 12 heads, 24 us (33 MB).  On the vector units the 32, the 16 and the 24 took 15.8, 47
// and 3.6 ms.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>

#include "it_latent.hpp"
#include "it_mfma.hpp"

namespace itkv {
namespace {  // each source that includes this compiles its own type's kernels
constexpr int kTile = 32;       // cached tokens
constexpr float kLazy = 8.0f;   // a maximum this much (log2) above the running one rescales; less waits
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) char lds_char;

template <int L, int R>
struct Tile {
  static constexpr int kRow = (L + R) * 2;            // bytes
  static constexpr int kChunks = kRow / 16;
  static constexpr int kBytes = kTile * kRow;
  // 16-byte chunk c of row r sits at chunk c ^ key(r) of it, such that sixteen rows'
  // same chunk, and eight rows' two neighbouring chunks, fall into different banks.
  // Rows of whole 128-byte lines: eight chunks are permuted.  Rows of an odd number of
  // half lines are 64 bytes further in the banks each, and four chunks are.
  static constexpr bool kLines = kChunks % 8 == 0;
  static_assert(kChunks % 4 == 0, "rows of whole 64 bytes");
  static __device__ __forceinline__ int key(int r) {
    return kLines ? ((r >> 1) & 3) << 1 | ((r >> 3) & 1) : ((r >> 2) & 1) << 1 | ((r >> 3) & 1);
  }
  // Loads of 64 chunks: kUnit rows are a whole number of them.
  static constexpr int kUnit = kLines ? 8 : 16;
  static constexpr int kUnitLoads = kUnit * kChunks / 64;
  static constexpr int kUnits = kTile / kUnit;
};
template <int L, int R, int QG, int KG>
struct Shape {
  static constexpr int kWaves = QG * KG, kThreads = 64 * kWaves;
  static constexpr int kFit = 144 * 1024 / (KG * Tile<L, R>::kBytes);
  static constexpr int kDepth = kFit < 1 ? 1 : kFit > 4 ? 4 : kFit;  // tiles of a token group
  static constexpr int kRing = KG * kDepth * Tile<L, R>::kBytes;
  static constexpr int kJoin = (KG - 1) * QG * 16 * L * 4;  // what token groups hand one another of O^T
  static constexpr int kLds = kRing > kJoin ? kRing : kJoin;
  static_assert(kLds <= 144 * 1024, "one workgroup per CU, and room for what is noted beside");
  // The loads of a tile, shared by QG waves: whole units, or parts of one (the last
  // part overlaps the one before where they do not divide).
  static constexpr int kUnitsOwn = QG < Tile<L, R>::kUnits ? Tile<L, R>::kUnits / QG : 1;
  static constexpr int kParts = QG > Tile<L, R>::kUnits ? QG / Tile<L, R>::kUnits : 1;
  static constexpr int kPart = (Tile<L, R>::kUnitLoads + kParts - 1) / kParts;
  static constexpr int kLoads = kUnitsOwn * kPart;  // of a wave
  static_assert(kDepth < 3 || kLoads * (kDepth - 2) < 64, "the counter of loads in flight");
  static_assert(kDepth > 1 || QG == 1, "one slot is one wave's own");
};

// The same value, of which nothing is known: what follows from it is computed where it is used,
// not kept in registers from loop turn to loop turn.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// A uniform element of a read-only array by a scalar load, which does not count among the vector loads.
__device__ __forceinline__ int scalar_at(const int32_t* p, int i) {
  return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}
// The same address in all lanes, so that it is kept in scalar registers.
__device__ __forceinline__ const char* uni(const char* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const char*>(uint64_t(uint32_t(uni(int(x >> 32)))) << 32 | uint32_t(uni(int(x))));
}
template <bool kNt>
__device__ __forceinline__ void load_lds(const char* base, uint32_t off, uint32_t m0) {
  if constexpr (kNt)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(m0), "v"(off), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m0), "v"(off), "s"(base) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 ld16_any(const uint16_t* p) {  // aligned to its elements
  uint4 x;
  __builtin_memcpy(&x, p, 16);
  return x;
}

typedef float v4f __attribute__((ext_vector_type(4)));
template <bool kBf16>
__device__ __forceinline__ v4f mfma16(const uint4& a, const uint4& b, const v4f& c) {
  if constexpr (kBf16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}
// Of a pair of 16-bit values: which are infinite or NaN (two bits); whether any of eight
// is; and the eight with those set to 0.
template <bool kBf16>
__device__ __forceinline__ uint32_t wild_halves(uint32_t x) {
  constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
  return uint32_t((x & kExp) == kExp) | uint32_t((x >> 16 & kExp) == kExp) << 1;
}
template <bool kBf16>
__device__ __forceinline__ bool any_wild(u32x4 v) {
  return (wild_halves<kBf16>(v[0]) | wild_halves<kBf16>(v[1]) | wild_halves<kBf16>(v[2]) | wild_halves<kBf16>(v[3])) != 0u;
}
template <bool kBf16>
__device__ __forceinline__ u32x4 cleaned(u32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t w = wild_halves<kBf16>(v[e]);
    v[e] &= ~((w & 1u ? 0xFFFFu : 0u) | (w & 2u ? 0xFFFF0000u : 0u));
  }
  return v;
}
// max / sum of x over the four lanes of a column: l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_quarters(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_halves(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}
__device__ __forceinline__ float sum_quarters(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_halves(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}

// What of a sequence a workgroup takes at a time.
struct Piece {
  int b;            // sequence
  int start, ctx;   // its visible tokens
  int steps;        // of KG tiles, of it
  int s0, n;        // the piece: steps s0 .. s0 + n
  int shared;       // workers from this one on that share the sequence
};
// x / d and x / d rounded up, 0 <= x < 2^21: the quotient of x + 1/2 is further from a whole
// number than its rounding reaches.
__device__ __forceinline__ int quotient(int x, int d) { return int((float(x) + 0.5f) * __builtin_amdgcn_rcpf(float(d))); }
__device__ __forceinline__ int over(int x, int d) { return quotient(x + d - 1, d); }

// How the steps of all sequences are divided among the workers; every wave finds it for
// itself from the lengths, sequences in chunks of 64, one a lane.
//   Runs: each worker takes `per` steps of all, which may begin and end inside sequences.
// Most workers then have two pieces, and a piece costs about as much as four steps beside
// its own: pages, queries and the first tile are waited for one after another, then sums are
// joined and stored.
//   Whole numbers of workers: sequences are divided, one piece a worker, where the longest
// piece is not four steps longer than a run.  For up to 64 sequences, which one chunk holds;
// more of them go by runs.
// Measured: 32 sequences of 256 to 8192 tokens, 32 heads, 41 us against 47 by runs; 24 of 100
// to 4096 with four drafted tokens of 12 heads, in workgroups of 64 queries, 27 against 37.
template <int KG>
struct Division {
  static constexpr int kPieceCost = 4;
  struct Span {
    int start, ctx, steps;
  };
  const LatentDecodeArgs& a;
  int per, total;
  bool whole;
  Span lanes;                 // of the chunk
  int chunk = 0, before = 0;  // and the steps before it

  __device__ __forceinline__ Span read(int c, bool latch) const {
    const int b = c + int(threadIdx.x & 63);
    const LatentSpan s = b < a.n_seqs ? latent_span(a, b, latch) : LatentSpan{0, 0};
    return {s.start, s.ctx, s.ctx > s.start ? ((s.ctx + kTile - 1) / kTile - s.start / kTile + KG - 1) / KG : 0};
  }
  static __device__ __forceinline__ int sum(int x) { return uni(__builtin_amdgcn_readlane(wave_inclusive_sum(x), 63)); }

  __device__ __forceinline__ Division(const LatentDecodeArgs& args, int workers, bool latch) : a(args) {
    lanes = read(0, latch);
    int mine = lanes.steps;
    for (int c = 64; c < a.n_seqs; c += 64) mine += read(c, latch).steps;
    total = sum(mine);
    per = max(1, (total + workers - 1) / workers);
    whole = false;
    if (a.n_seqs > 64 || total >= 1 << 20) return;
    const int busy = __popcll(__ballot(lanes.steps > 0));
    if (busy == 0 || busy >= workers) return;
    for (int length = per; length <= per + kPieceCost; ++length) {  // of a piece at most
      if (sum(over(lanes.steps, length)) > workers) continue;
      per = length;
      whole = true;
      return;
    }
  }
  // The piece that worker w takes of a division into whole numbers; n 0: none.
  __device__ __forceinline__ Piece of(int w) const {
    const int mine = over(lanes.steps, per), upto = wave_inclusive_sum(mine);
    const uint64_t past = __ballot(w < upto);
    if (past == 0) return {};
    const int i = __builtin_ctzll(past), steps = __builtin_amdgcn_readlane(lanes.steps, i), n = __builtin_amdgcn_readlane(mine, i);
    const int first = __builtin_amdgcn_readlane(upto, i) - n, j = w - first;
    const int each = uni(quotient(steps, n)), more = steps - each * n;
    return {uni(i), __builtin_amdgcn_readlane(lanes.start, i), __builtin_amdgcn_readlane(lanes.ctx, i), steps,
            uni(j * each + min(j, more)), uni(each + (j < more)), uni(n)};
  }
  // The piece that begins at step t of all, in worker w's run, which ends at `end`; t does not
  // decrease from call to call.
  __device__ __forceinline__ Piece at(int t, int end, int w) {
    for (;;) {  // ends: t is below the total
      const int upto = before + wave_inclusive_sum(lanes.steps), all = __builtin_amdgcn_readlane(upto, 63);
      if (t >= all) {
        before = uni(all);
        chunk += 64;
        lanes = read(chunk, false);
        continue;
      }
      const int i = __builtin_ctzll(__ballot(t < upto)), steps = __builtin_amdgcn_readlane(lanes.steps, i);
      const int last = __builtin_amdgcn_readlane(upto, i), s0 = t - (last - steps);
      return {uni(chunk + i), __builtin_amdgcn_readlane(lanes.start, i), __builtin_amdgcn_readlane(lanes.ctx, i), steps,
              uni(s0), uni(min(end - t, steps - s0)), uni((last - 1) / per - w + 1)};
    }
  }
};

template <bool kBf16, int L, int R, int QG, int KG, bool kNt>
__global__ __launch_bounds__(64 * QG * KG, QG * KG > 4 ? 2 : 1) void latent_decode_split(LatentDecodeArgs a, LatentSplitPlan plan) {
  using T = Tile<L, R>;
  using S = Shape<L, R, QG, KG>;
  constexpr int kDepth = S::kDepth, ND = L / 16, NQ = (L + R) / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float2 ml_of[S::kWaves][16];
  __shared__ uint32_t wild_of[S::kWaves][ND / 8][64];  // of a lane's results, which a drafted token's infinities and NaN reach
  const int lane = int(threadIdx.x & 63), wave = uni(int(threadIdx.x >> 6)), quarter = lane >> 4, col = lane & 15;
  const int qg = wave % QG, kg = wave / QG;
  // The workgroups that share a run's tiles on one XCD, next to one another.
  const int id = int(blockIdx.x), slot = id >> 3, worker = slot / plan.row_wgs * 8 + (id & 7), rw = slot % plan.row_wgs;
  if (worker >= plan.workers) return;
  Division<KG> division(a, plan.workers, id == 0 && wave == 0);
  int t = uni(worker * division.per);
  const int t_end = division.whole ? t + 1 : uni(min(division.total, t + division.per));
  if (!division.whole && t >= t_end) return;

  // This lane's query.
  const int rows = a.q_len * a.n_heads, row = (rw * QG + qg) * 16 + col;
  const bool live = row < rows;
  const int tok = live ? row / a.n_heads : a.q_len - 1, head = live ? row - tok * a.n_heads : 0;

  // LDS addresses.  For Q K^T: row `col` (+ 16), chunk 4 k + quarter.  For C^T: row 4
  // quarter + j / 4 (+ 16), values 4 (j % 4) .. of a d-tile's 16, j = lane % 16.  What
  // the swizzle lets be an instruction's offset is left out.
  const uint32_t ring = lds_off(lds) + uint32_t(kg * kDepth * T::kBytes);
  constexpr int kQkBases = T::kLines ? 2 : 1, kPvBases = 2 * kQkBases;
  uint32_t qk_at[kQkBases], pv_at[kPvBases];
#pragma unroll
  for (int b = 0; b < kQkBases; ++b) qk_at[b] = ring + uint32_t(col * T::kRow + (((4 * b + quarter) ^ T::key(col)) << 4));
#pragma unroll
  for (int b = 0; b < kPvBases; ++b) {
    const int j = lane & 15, r = 4 * quarter + (j >> 2), c = 2 * b + ((j & 3) >> 1);
    pv_at[b] = ring + uint32_t(r * T::kRow + ((c ^ T::key(r)) << 4) + 8 * (j & 1));
  }
  // The wave's loads of a tile.
  const int unit0 = S::kParts > 1 ? qg / S::kParts : qg * S::kUnitsOwn;
  const int load0 = S::kParts > 1 ? min(qg % S::kParts * S::kPart, T::kUnitLoads - S::kPart) : 0;

  while (t < t_end) {
    const Piece found = division.whole ? division.of(worker) : division.at(t, t_end, worker);
    const Piece pc = {uni(found.b), uni(found.start), uni(found.ctx), uni(found.steps), uni(found.s0), uni(found.n), uni(found.shared)};
    const int s0 = pc.s0, n_steps = pc.n;
    if (n_steps == 0) return;
    t = division.whole ? t_end : uni(t + n_steps);
    if (s0 == 0 && rw == 0 && threadIdx.x == 0) plan.shares[pc.b] = make_int2(worker, pc.shared);
    const int32_t* const bt = a.bt + int64_t(pc.b) * a.max_blocks;
    const int tile0 = pc.start / kTile + s0 * KG + kg;  // this wave's first tile
    const int tiles = max(0, min(n_steps, ((pc.ctx + kTile - 1) / kTile - tile0 + KG - 1) / KG));

    // The pages of tile i's eight-token runs that this wave loads, read a tile ahead by
    // scalar loads that wait for one another no longer than for one.  Tokens outside
    // [start, ctx) are read from the nearest page that is held, and masked.
    constexpr int kRuns = S::kUnitsOwn * T::kUnit / 8;
    const auto key_of = [&](int i, int run) __attribute__((always_inline)) {
      const int key = (tile0 + i * KG) * kTile + unit0 * T::kUnit + 8 * run;
      return uni(min(max(key, pc.start & ~7), (pc.ctx - 1) & ~7));
    };
    constexpr int kFirst = kDepth > 1 ? kDepth - 1 : 1;  // tiles whose pages are read together at first
    int ids[kRuns], first_ids[kFirst][kRuns];
    const auto read_ids = [&](int i, int (&to)[kRuns]) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < kRuns; ++r) to[r] = scalar_at(bt, key_of(i, r) >> a.log2_bs);
    };
#pragma unroll
    for (int i = 0; i < kFirst; ++i) read_ids(i, first_ids[i]);
    // Tile i of this wave into ring slot i % kDepth: this wave's share of its loads.
    const auto issue = [&](int i, const int (&ids)[kRuns]) __attribute__((always_inline)) {
      const uint32_t m0 = ring + uint32_t((kDepth == 1 ? 0 : i % kDepth) * T::kBytes);
      const char* pages[kRuns];
      bool bad = false;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const int k = key_of(i, r), id = uni(ids[r]);
        const bool off = id < 0 || id >= a.num_blocks;  // uniform
        bad |= off;
        pages[r] = uni(a.pool + int64_t(off ? 0 : id) * a.page_bytes + (k & ((1 << a.log2_bs) - 1)) * T::kRow);
      }
      if (bad && lane == 0) atomicOr(a.err, kErrBlock);
      // This lane's chunks of a unit's rows, as the loads place them: where registers are short,
      // computed for each tile.
      const int ln = L > 256 && S::kWaves > 4 ? fresh(lane) : lane;
      uint32_t from[S::kPart];
#pragma unroll
      for (int j = 0; j < S::kPart; ++j) {
        const int p = 64 * (load0 + j) + ln, r = p / T::kChunks, c = (p - r * T::kChunks) ^ T::key(r);
        from[j] = uint32_t(r * T::kRow + c * 16);
      }
#pragma unroll
      for (int u = 0; u < S::kUnitsOwn; ++u) {
        const int unit = unit0 + u;
        const uint32_t to = m0 + uint32_t((unit * T::kUnitLoads + load0) * 1024);
        if constexpr (T::kLines) {
          const char* const base = pages[u];
          const uint32_t flip = (unit & 1) << 4;  // the rows' key has bit 0 of the unit's number
#pragma unroll
          for (int j = 0; j < S::kPart; ++j) load_lds<kNt>(base, from[j] ^ flip, uni(to + uint32_t(j * 1024)));
        } else {  // sixteen rows are two runs of eight; the load in the middle has rows of both
          const char* const first = pages[2 * u];
          const char* const second = pages[2 * u + 1] - 8 * T::kRow;
#pragma unroll
          for (int j = 0; j < S::kPart; ++j) {
            const int at = load0 + j;  // uniform
            if (2 * at + 1 != T::kUnitLoads) load_lds<kNt>(2 * at < T::kUnitLoads ? first : second, from[j], uni(to + uint32_t(j * 1024)));
            else dma_b128((from[j] < 8u * T::kRow ? first : second) + from[j], uni(to + uint32_t(j * 1024)));
          }
        }
      }
    };
    if constexpr (kDepth > 1) {
#pragma unroll 1
      for (int i = 0; i < kDepth - 1 && i < tiles; ++i) {
#pragma unroll
        for (int r = 0; r < kRuns; ++r) ids[r] = i == 0 ? first_ids[0][r] : i == 1 ? first_ids[kFirst > 1 ? 1 : 0][r] : first_ids[kFirst > 2 ? 2 : 0][r];
        issue(i, ids);
      }
      read_ids(kDepth - 1, ids);  // past the last tile: the last page again
    } else {
#pragma unroll
      for (int r = 0; r < kRuns; ++r) ids[r] = first_ids[0][r];
    }

    uint4 q[NQ];
    {
      const int64_t at = int64_t(pc.b) * a.q_len + tok;
      const uint16_t* const ql = static_cast<const uint16_t*>(a.q_latent) + at * a.ql_stride + head * a.ql_head + 8 * quarter;
      const uint16_t* const qr = static_cast<const uint16_t*>(a.q_rope) + at * a.qr_stride + head * a.qr_head + 8 * quarter;
#pragma unroll
      for (int i = 0; i < L / 32; ++i) q[i] = ld16_any(ql + 32 * i);
#pragma unroll
      for (int i = 0; i < R / 32; ++i) q[L / 32 + i] = ld16_any(qr + 32 * i);
      // Waited for here: at their first use, inside the loop, every turn would wait again, for
      // the tiles in flight too.
      if constexpr (S::kWaves > 4) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          u32x4 x = __builtin_bit_cast(u32x4, q[i]);
          asm volatile("" : "+v"(x));
          q[i] = __builtin_bit_cast(uint4, x);
        }
      }
    }
    v4f o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v4f{};
    float m_run = -INFINITY, l_run = 0.0f;
    bool wild = false;
    for (int d = 0; d < ND / 8; ++d) wild_of[wave][d][lane] = 0u;
    // The end of a step's last tile, of whichever token group.
    const auto step_end = [&](int i) { return (pc.start / kTile + (s0 + i + 1) * KG) * kTile; };

    const auto compute = [&](int i) __attribute__((always_inline)) {
      const int key0 = (tile0 + i * KG) * kTile;
      const uint32_t at = kDepth == 1 ? 0u : uint32_t(i % kDepth) * T::kBytes;
      // This tile's bases, made opaque: all else of an address is an offset in its instruction.
      uint32_t qk_base[kQkBases], pv_base[kPvBases];
#pragma unroll
      for (int b = 0; b < kQkBases; ++b) {
        qk_base[b] = qk_at[b] + at;
        asm volatile("" : "+v"(qk_base[b]));
      }
#pragma unroll
      for (int b = 0; b < kPvBases; ++b) {
        pv_base[b] = pv_at[b] + at;
        asm volatile("" : "+v"(pv_base[b]));
      }
      // The operands of kAhead steps are on their way while one is multiplied; the
      // scheduler, left to itself, loads so far ahead that it runs out of registers.
      constexpr int kAhead = L > 256 && S::kWaves > 4 ? 1 : 4;
      v4f s[2] = {v4f{}, v4f{}};
      uint4 key_rows[kAhead + 1][2];
      const auto load_rows = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const lds_char* const p = reinterpret_cast<const lds_char*>(uintptr_t(qk_base[k % kQkBases])) + k / kQkBases * (64 * kQkBases) + u * 16 * T::kRow;
          key_rows[k % (kAhead + 1)][u] = __builtin_bit_cast(uint4, *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(p));
        }
      };
#pragma unroll
      for (int k = 0; k < kAhead; ++k) load_rows(k);
#pragma unroll
      for (int k = 0; k < NQ; ++k) {
        if (k + kAhead < NQ) load_rows(k + kAhead);
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = mfma16<kBf16>(key_rows[k % (kAhead + 1)][u], q[k], s[u]);
        __builtin_amdgcn_sched_barrier(0);
      }
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * a.scale_log2;
      const bool edge = key0 < pc.start || key0 + kTile > pc.ctx - a.q_len + 1;  // uniform
      if (edge) {
        const int lo = pc.start - key0, hi = pc.ctx - a.q_len + 1 + tok - key0, first = fresh(lane) >> 4 << 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = 16 * (e >> 2) + first + (e & 3);
          x[e] = r >= lo && r < hi ? x[e] : -INFINITY;
        }
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      top = max_quarters(top);
      if (__ballot(top > m_run + kLazy) != 0) {  // uniform, rare after the first tile
        const float m_new = fmaxf(m_run, top);
        const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][e] *= alpha;
        m_run = m_new;
      }
      const float use = m_run == -INFINITY ? 0.0f : m_run;
      // P rounded to the rows' type, and summed as rounded: numerator and denominator hold the same weights.
      uint32_t p[4];
      const uint32_t ones = kBf16 ? 0x3F803F80u : 0x3C003C00u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = pack2<kBf16>(__builtin_amdgcn_exp2f(x[2 * e] - use), __builtin_amdgcn_exp2f(x[2 * e + 1] - use));
        l_run = dot2_ones<kBf16>(p[e], l_run, ones);
      }
      const uint4 weights = make_uint4(p[0], p[1], p[2], p[3]);
      const auto values = [&](int d, int u) __attribute__((always_inline)) {
        lds_char* const v = reinterpret_cast<lds_char*>(uintptr_t(pv_base[d % kPvBases])) + d / kPvBases * (32 * kPvBases) + u * 16 * T::kRow;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(v)));
      };
      // A weight of 0 does not silence an infinity.  Rows that no query sees are cleared in
      // LDS, by each wave for itself (others may still be scoring them: those scores are
      // masked).  Of a drafted token's rows, which earlier tokens do not see, infinities and
      // NaN are cleared, once all have scored them, and noted for the queries that see them.
      const bool drafted = a.q_len > 1 && step_end(i) > pc.ctx - a.q_len + 1;  // the same in all waves
      const int lo = max(pc.start - key0, 0), hi = min(pc.ctx - key0, kTile), late = max(lo, pc.ctx - a.q_len + 1 - key0);
      const auto chunk = [&](int r) __attribute__((always_inline)) {  // a row's values, 16 bytes a lane
        return reinterpret_cast<__attribute__((address_space(3))) u32x4*>(uintptr_t(ring + at + uint32_t(r * T::kRow + fresh(lane) * 16)));
      };
      if (drafted) {
        const int seen = pc.ctx - a.q_len + 1 + tok - key0;
#pragma unroll 1
        for (int r = late; r < hi; ++r) {
          const lds_char* const at_row = reinterpret_cast<const lds_char*>(uintptr_t(ring + at + uint32_t(r * T::kRow)));
          if (__ballot(lane < L / 8 && any_wild<kBf16>(*chunk(r))) == 0) continue;  // uniform, nearly always
#pragma unroll 1
          for (int d = 0; d < ND; ++d) {  // values 16 d + 4 quarter ..
            const int c = 2 * d + (quarter >> 1);
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x2*>(at_row + ((c ^ T::key(r)) << 4) + 8 * (quarter & 1));
            const uint32_t bits = wild_halves<kBf16>(v[0]) | wild_halves<kBf16>(v[1]) << 2;
            if (r < seen) wild_of[wave][d / 8][lane] |= bits << (d % 8 * 4);
          }
          wild = true;
        }
        if constexpr (QG > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      if (edge) {
#pragma unroll 1
        for (int r = 0; r < kTile; ++r) {
          if (lane >= L / 8) continue;
          if (r < lo || r >= hi) {
            *chunk(r) = u32x4{};
          } else if (r >= late && drafted) {
            const u32x4 v = *chunk(r);
            if (any_wild<kBf16>(v)) *chunk(r) = cleaned<kBf16>(v);
          }
        }
      }
      {
        constexpr int kNext = L > 256 && S::kWaves > 4 ? 3 : ND < 8 ? ND : 8;  // d-tiles ahead
        uint2 v[kNext + 1][2];
#pragma unroll
        for (int d = 0; d < kNext; ++d) v[d][0] = values(d, 0), v[d][1] = values(d, 1);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          if (d + kNext < ND) v[(d + kNext) % (kNext + 1)][0] = values(d + kNext, 0), v[(d + kNext) % (kNext + 1)][1] = values(d + kNext, 1);
          const uint2 v0 = v[d % (kNext + 1)][0], v1 = v[d % (kNext + 1)][1];
          o[d] = mfma16<kBf16>(make_uint4(v0.x, v0.y, v1.x, v1.y), weights, o[d]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };

    if constexpr (kDepth == 1) {
      for (int i = 0; i < tiles; ++i) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile before is read
        issue(i, ids);
        read_ids(i + 1, ids);
        wait_loads<0>();
        compute(i);
      }
    } else {
      const int turns = QG == 1 ? tiles : n_steps;  // waves that share tiles pass the same barriers
      for (int i = 0; i < turns; ++i) {
        // Tile i has arrived when no more loads are in flight than those issued after it.
        const int ahead = min(tiles - 1 - i, kDepth - 2);
        if (kDepth > 3 && ahead >= 2) wait_loads<2 * S::kLoads>();
        else if (kDepth > 2 && ahead == 1) wait_loads<S::kLoads>();
        else wait_loads<0>();
        if constexpr (QG == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (i + kDepth - 1 < tiles) issue(i + kDepth - 1, ids);  // where tile i - 1 was
        read_ids(i + kDepth, ids);
        if (i < tiles) compute(i);
        else if (QG > 1 && a.q_len > 1 && step_end(i) > pc.ctx - a.q_len + 1) asm volatile("s_barrier" ::: "memory");  // compute()'s
      }
    }
    float l = sum_quarters(l_run), M = m_run;
    if (wild) {  // uniform
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const uint32_t bits = wild_of[wave][d / 8][lane] >> (d % 8 * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] = bits >> e & 1u ? NAN : o[d][e];
      }
    }

    // The token groups joined, each for a part of the values.
    constexpr int kOwn = ND / KG;
    v4f own[kOwn];
    if constexpr (KG > 1) {
      if (quarter == 0) ml_of[wave][col] = make_float2(m_run, l);
      __syncthreads();  // all tiles are read too
      l = 0.0f;
#pragma unroll
      for (int g = 0; g < KG; ++g) M = fmaxf(M, ml_of[g * QG + qg][col].x);
      const float use = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const float2 x = ml_of[g * QG + qg][col];
        l = fmaf(__builtin_amdgcn_exp2f(x.x - use), x.y, l);
      }
      const float mine = __builtin_amdgcn_exp2f(m_run - use);
      // Token group kg keeps d-tiles kg ND / KG ..: it writes the others' and reads theirs.
      v4f* const join = reinterpret_cast<v4f*>(lds);
      const auto place = [&](int from, int to, int d) { return (((from * (KG - 1) + to - (to > from)) * QG + qg) * kOwn + d) * 64 + lane; };
      if constexpr (KG == 2) {
#pragma unroll
        for (int d = 0; d < kOwn; ++d) {
          const v4f x = o[d] * mine, y = o[kOwn + d] * mine;
          join[place(kg, 1 - kg, d)] = kg ? x : y;
          own[d] = kg ? y : x;
        }
      } else {
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          if (g == kg) continue;  // uniform
#pragma unroll
          for (int d = 0; d < kOwn; ++d) join[place(kg, g, d)] = o[g * kOwn + d] * mine;
        }
#pragma unroll
        for (int g = 0; g < KG; ++g)
          if (g == kg) {
#pragma unroll
            for (int d = 0; d < kOwn; ++d) own[d] = o[g * kOwn + d] * mine;
          }
      }
      __syncthreads();
#pragma unroll
      for (int g = 1; g < KG; ++g)
#pragma unroll
        for (int d = 0; d < kOwn; ++d) own[d] += join[place((kg + g) % KG, kg, d)];
    } else {
#pragma unroll
      for (int d = 0; d < kOwn; ++d) own[d] = o[d];
    }
    if (n_steps == pc.steps) {  // the whole sequence: done
      if (live) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t out = ((int64_t(pc.b) * a.q_len + tok) * a.n_heads + head) * L + 16 * kOwn * kg + 4 * quarter;
#pragma unroll
        for (int d = 0; d < kOwn; ++d) {
          const v4f x = own[d] * inv;
          if (a.out_dtype == IT_F32) *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + out + 16 * d) = x;
          else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + out + 16 * d) = make_uint2(pack2<kBf16>(x[0], x[1]), pack2<kBf16>(x[2], x[3]));
        }
      }
    } else {  // slot 1: the piece that begins its sequence; 0: one that continues it
      const int64_t part = ((int64_t(worker) * plan.row_wgs + rw) * 2 + (s0 == 0)) * QG + qg;
      v4f* const to = reinterpret_cast<v4f*>(plan.o) + part * (ND * 64) + kOwn * kg * 64 + lane;
#pragma unroll
      for (int d = 0; d < kOwn; ++d) __builtin_nontemporal_store(own[d], to + d * 64);  // on its way at once, not at the kernel's end
      if (kg == 0 && quarter == 0) plan.ml[part * 16 + col] = make_float2(M, l);
    }
    __syncthreads();  // before the next piece's loads into the ring, and ml_of
  }
}

// Joins the pieces of sequences that several workgroups shared, and zeroes rows of
// empty ones.  grid: (four d-tiles, 16 queries, sequence); a wave takes a d-tile.
template <bool kBf16, int QG, int KG>
__global__ __launch_bounds__(256) void latent_decode_join(LatentDecodeArgs a, LatentSplitPlan plan) {
  const int lane = int(threadIdx.x & 63), quarter = lane >> 4, col = lane & 15;
  const int nd = int(gridDim.x) * 4, dt = int(blockIdx.x) * 4 + int(threadIdx.x >> 6), group = int(blockIdx.y), b = int(blockIdx.z);
  const int rw = group / QG, qg = group - rw * QG;
  // A sequence that holds something has been given its first worker; what others hold is of an earlier call.
  const LatentSpan span = latent_span(a, b, false);
  const int2 share = plan.shares[b];
  const bool some = uni(span.ctx) > uni(span.start);
  const int w0 = uni(share.x), w1 = w0 + uni(share.y) - 1;
  if (some && w0 == w1) return;  // one workgroup wrote it
  const int rows = a.q_len * a.n_heads, row = group * 16 + col;
  v4f sum = v4f{};
  float inv = 0.0f;
  if (some) {
    const auto part = [&](int w) { return ((int64_t(w) * plan.row_wgs + rw) * 2 + (w == w0)) * QG + qg; };
    float M = -INFINITY, l = 0.0f;
    // Pieces eight at a time, their maxima, sums and values loaded together.
    constexpr int kAtOnce = 8;
#pragma unroll 1
    for (int w = w0; w <= w1; w += kAtOnce) {
      float2 ml[kAtOnce];
      v4f x[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int64_t from = part(min(w + i, w1));
        ml[i] = plan.ml[from * 16 + col];
        x[i] = reinterpret_cast<const v4f*>(plan.o)[(from * nd + dt) * 64 + lane];
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
      const float use = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(M - use);
      l *= old;
      sum *= old;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i].x - use);
        if (w + i > w1) continue;  // uniform
        l = fmaf(f, ml[i].y, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, x[i][e], sum[e]);
      }
      M = top;
    }
    inv = l == 0.0f ? 0.0f : 1.0f / l;
  }
  if (row >= rows) return;
  const int64_t out = (int64_t(b) * rows + row) * (nd * 16) + 16 * dt + 4 * quarter;
  sum *= inv;
  if (a.out_dtype == IT_F32) *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + out) = sum;
  else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + out) = make_uint2(pack2<kBf16>(sum[0], sum[1]), pack2<kBf16>(sum[2], sum[3]));
}

template <bool kBf16, int L, int R, int QG, int KG, bool kNt>
hipError_t launch_split(const LatentDecodeArgs& a, const LatentSplitPlan& p, hipStream_t s) {
  static std::atomic<uint64_t> opted{0};
  using S = Shape<L, R, QG, KG>;
  auto* const kern = latent_decode_split<kBf16, L, R, QG, KG, kNt>;
  if (const hipError_t e = opt_in_lds(reinterpret_cast<const void*>(kern), S::kLds, opted); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3(unsigned((p.workers + 7) / 8 * 8 * p.row_wgs)), dim3(S::kThreads), S::kLds, s, a, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid(L / 64, unsigned((a.q_len * a.n_heads + 15) / 16), unsigned(a.n_seqs));
  hipLaunchKernelGGL((latent_decode_join<kBf16, QG, KG>), grid, dim3(256), 0, s, a, p);
  return hipGetLastError();
}
// Where several workgroups read a tile, the later ones find it in their XCD's L2 (128 heads over
// 64 x 1000 tokens 49 us, 53 past it); else tiles go past it.
template <bool kBf16, int L, int R, int QG, int KG>
hipError_t launch_groups(const LatentDecodeArgs& a, const LatentSplitPlan& p, hipStream_t s) {
  return p.row_wgs == 1 ? launch_split<kBf16, L, R, QG, KG, true>(a, p, s) : launch_split<kBf16, L, R, QG, KG, false>(a, p, s);
}
template <bool kBf16, int L, int R>
hipError_t launch(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s) {
  if (qg == 1) return launch_groups<kBf16, L, R, 1, 4>(a, p, s);
  if constexpr (L + R <= kLatentNarrow) return launch_groups<kBf16, L, R, 2, 4>(a, p, s);
  else if (qg == 2) return launch_groups<kBf16, L, R, 2, 2>(a, p, s);
  else if (qg == 4) return launch_groups<kBf16, L, R, 4, 1>(a, p, s);
  else return launch_groups<kBf16, L, R, 8, 1>(a, p, s);
}
template <bool kBf16>
hipError_t launch_latent_decode(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s) {
  if (a.latent == 512) return launch<kBf16, 512, 64>(a, p, qg, s);
  if (a.latent == 128) return launch<kBf16, 128, 64>(a, p, qg, s);
  return a.rope == 64 ? launch<kBf16, 256, 64>(a, p, qg, s) : launch<kBf16, 256, 32>(a, p, qg, s);
}
}  // namespace
}  // namespace itkv
