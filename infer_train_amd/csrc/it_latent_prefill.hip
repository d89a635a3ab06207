// it_latent_prefill.hip -- expanded latent attention on the matrix cores: keys of
// a part per head and a rope part that all heads share, values of another width,
// contiguous and per head (F16 and BF16, the usual widths).
//
// One workgroup = (sequence, head, 128 queries), four waves of 32 queries each; two
// workgroups per CU, each with its own phase, so that one's softmax runs beside the
// other's products.  Per block of 64 keys, staged in LDS by direct loads (two
// blocks of it: one is read while the next arrives):
//   S^T = K Q^T    v_mfma_f32_32x32x16, keys are its rows, queries its columns, so a
//                  lane owns one query: its maximum and sum are in-lane plus a swap
//                  with lane ^ 32; the key's two parts are two runs of products;
//   O^T += V^T P^T the probabilities go back into operands straight from the S^T
//                  registers; V^T comes transposed out of LDS (ds_read_b64_tr_b16).
// Online softmax in fp32, the maximum raised only when it grew by more than 2^8.
// Rows of a part are 16, 8 or 4 chunks of 16 bytes, XOR-swizzled by row so that the
// operand reads are free of bank conflicts.
// Bound by LDS reads and products in turn: per block a wave takes 24 KB of keys at 128
// bytes a clock and 16 KB of values at 64, 450 clocks of the CU, 8 waves 3600, where
// their 320 products take 2560 of the four matrix cores, and the two overlap by half.
// Eight chunks of 512 queries over 1536 to 2560 keys, 32 heads of 192 and 128 elements in
// bf16: 196 us (192 to 201 from run to run), 761 TFLOP/s of the 1317 that an 8192^3 product reaches (on the vector
// units 113 ms).  Blocks of 32 keys take 4% longer, and where they let three waves on a SIMD
// (25 registers spilled) 90%; the scale in the exponent's fma, the reads ordered ahead of
// the products, and wave priorities are all within 2%.
#include <hip/hip_runtime.h>

#include <atomic>

#include "it_latent.hpp"
#include "it_mfma.hpp"

using namespace itkv;

namespace {
constexpr int kQ = 32;              // queries of a wave
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kQueries = kQ * kWaves;
constexpr int kKeys = 64;           // of a block
constexpr float kLazy = 8.0f;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// 64 rows of D elements in LDS.
template <int D>
struct Part {
  static constexpr int kRow = D * 2, kChunks = kRow / 16, kBytes = kKeys * kRow;
  static_assert(kChunks == 16 || kChunks == 8 || kChunks == 4, "");
  // Chunk c of row r sits at c ^ key(r): of sixteen rows the same chunk, and of four rows four
  // neighbouring ones, fall into different banks (rows of 128 and 64 bytes are shifted against
  // one another by themselves).
  static __device__ __forceinline__ int key(int r) {
    return kChunks == 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : kChunks == 8 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3;
  }
  static constexpr int kLoads = kBytes / 1024 / kWaves;  // of a wave
  static constexpr int kRows = 64 / kChunks;             // of a load
  // A wave's loads of the rows from `base`, `stride` bytes apart, those past `last` read again.
  static __device__ __forceinline__ void load(const char* base, uint32_t stride, int last, uint32_t lds, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = (wave * kLoads + j) * kRows + lane / kChunks, c = lane % kChunks ^ key(r);
      const uint32_t from = uint32_t(min(r, last)) * stride + uint32_t(c * 16);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uni(lds + uint32_t((wave * kLoads + j) * 1024))), "v"(from),
                   "s"(base)
                   : "memory", "m0");
    }
  }
};

template <bool kBf16>
__device__ __forceinline__ uint32_t wild_halves(uint32_t x) {  // which of a pair are infinite or NaN
  constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
  return uint32_t((x & kExp) == kExp) | uint32_t((x >> 16 & kExp) == kExp) << 1;
}

// Half f of it as fp32.
template <bool kBf16>
__device__ __forceinline__ float half_value(uint32_t x, int f) {
  const uint32_t bits = f ? x >> 16 : x & 0xFFFFu;
  return kBf16 ? __uint_as_float(bits << 16) : float(__builtin_bit_cast(_Float16, uint16_t(bits)));
}

template <bool kBf16, int DN, int R, int DV>
__global__ __launch_bounds__(kThreads, 2) void latent_prefill(LatentPrefillArgs a, int n_qb) {
  using K = Part<DN>;
  using KR = Part<R>;
  using V = Part<DV>;
  constexpr int ND = DV / 32, kStage = K::kBytes + KR::kBytes + V::kBytes;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = int(threadIdx.x & 63), wave = uni(int(threadIdx.x >> 6)), h = lane >> 5, col = lane & 31;
  // All query blocks of a (sequence, head) on one XCD, whose L2 then holds its keys; the longest first.
  const int id = int(blockIdx.x), slot = id >> 3, pair = slot / n_qb * 8 + (id & 7), qb = n_qb - 1 - slot % n_qb;
  const int b = pair / a.n_heads, head = pair - b * a.n_heads;
  if (b >= a.n_seqs) return;
  const int q0 = uni(a.cu_q[b]), q1 = uni(a.cu_q[b + 1]), k0 = uni(a.cu_k[b]), k1 = uni(a.cu_k[b + 1]);
  if (!latent_prefill_fits(a, q0, q1, k0, k1)) return;
  const int nq = q1 - q0, n = k1 - k0;
  if (qb * kQueries >= nq) return;
  // Query i sees the keys before limit(i).
  const auto limit = [&](int i) { return a.causal ? min(n, max(0, n - nq + i + 1)) : n; };
  const int first = qb * kQueries, row = first + wave * kQ + col;
  const int mine = limit(row < nq ? row : nq - 1);                                       // of this lane's query
  const int wave_lo = uni(limit(min(first + wave * kQ, nq - 1))), wave_hi = uni(limit(min(first + wave * kQ + kQ, nq) - 1));
  const int lo = uni(limit(first)), hi = uni(limit(min(first + kQueries, nq) - 1));      // of the workgroup's
  const int blocks = (hi + kKeys - 1) / kKeys;

  const int64_t es = 2;
  const char* const k_at = static_cast<const char*>(a.k) + (int64_t(k0) * a.k_stride + head * a.k_head) * es;
  const char* const v_at = static_cast<const char*>(a.v) + (int64_t(k0) * a.v_stride + head * a.v_head) * es;
  const char* const r_at = static_cast<const char*>(a.k_rope) + int64_t(k0) * a.rope_stride * es;
  const uint32_t ring = lds_off(lds);
  const auto issue = [&](int i) __attribute__((always_inline)) {
    const uint32_t at = ring + uint32_t((i & 1) * kStage);
    const int last = n - 1 - i * kKeys;
    K::load(k_at + int64_t(i * kKeys) * a.k_stride * es, uint32_t(a.k_stride * es), last, at, wave, lane);
    KR::load(r_at + int64_t(i * kKeys) * a.rope_stride * es, uint32_t(a.rope_stride * es), last, at + K::kBytes, wave, lane);
    V::load(v_at + int64_t(i * kKeys) * a.v_stride * es, uint32_t(a.v_stride * es), last, at + K::kBytes + KR::kBytes, wave, lane);
  };
  if (blocks > 0) issue(0);

  uint4 q[(DN + R) / 16];
  {
    const uint16_t* const at = static_cast<const uint16_t*>(a.q) + int64_t(q0 + min(row, nq - 1)) * a.q_stride + head * a.q_head + 8 * h;
#pragma unroll
    for (int i = 0; i < (DN + R) / 16; ++i) __builtin_memcpy(&q[i], at + 16 * i, 16);
  }
  v16f o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = v16f{};
  float m_run = -INFINITY, l_run = 0.0f;

  // LDS addresses of the operands: chunk 2 k + h of key row `col`; of the values rows 4 h +
  // j / 4 (+ 8 g + 16 t), columns 16 (lane / 16 % 2) + 4 (j % 4) of a d-tile, j = lane % 16.
  const uint32_t k_key = uint32_t(K::key(col)), r_key = uint32_t(KR::key(col));
  const int j16 = lane & 15, v_row = 4 * h + (j16 >> 2), v_chunk = 2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1);

#pragma unroll 1
  for (int i = 0; i < blocks; ++i) {
    // Block i is there, and all waves have done with the one before.
    asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (i + 1 < blocks) issue(i + 1);
    const int key0 = i * kKeys;
    const uint32_t stage = ring + uint32_t((i & 1) * kStage), v_stage = stage + K::kBytes + KR::kBytes;
    // Values of rows past the last key are cleared, since a weight of 0 does not silence an
    // infinity.  Infinities and NaN of others that not every query of the workgroup sees are added
    // to the results of the queries that do, then cleared.  Each wave looks at all rows for itself:
    // two workgroups leave no LDS for a word between them.
    const int end = min(n - key0, kKeys), late = max(0, lo - key0);
    bool wild = false;  // uniform, the same in all waves, and nearly never
    if (key0 + kKeys > lo) {  // uniform
      bool any = false;
      for (int c = lane; c < kKeys * V::kChunks; c += 64) {
        const int r = c / V::kChunks;
        lds_u32x4* const at = reinterpret_cast<lds_u32x4*>(uintptr_t(v_stage + uint32_t(c * 16)));
        if (r >= end) {
          *at = u32x4{};
        } else if (r >= late) {
          const u32x4 x = *at;
          any |= (wild_halves<kBf16>(x[0]) | wild_halves<kBf16>(x[1]) | wild_halves<kBf16>(x[2]) | wild_halves<kBf16>(x[3])) != 0u;
        }
      }
      wild = __ballot(any) != 0;
    }
    const auto clean = [&]() __attribute__((always_inline)) {  // once all waves have read them
      __syncthreads();
      for (int c = int(threadIdx.x); c < kKeys * V::kChunks; c += kThreads) {
        if (c / V::kChunks < late) continue;
        lds_u32x4* const at = reinterpret_cast<lds_u32x4*>(uintptr_t(v_stage + uint32_t(c * 16)));
        u32x4 x = *at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = wild_halves<kBf16>(x[e]);
          x[e] &= ~((w & 1u ? 0xFFFFu : 0u) | (w & 2u ? 0xFFFF0000u : 0u));
        }
        *at = x;
      }
      __syncthreads();
    };
    const bool idle = key0 >= wave_hi;  // uniform: nothing here for this wave's queries
    // The block's scores of this lane's query, and the largest of all of them.
    const auto score = [&](float (&x)[2][16]) __attribute__((always_inline)) {
      uint32_t k_base = stage + uint32_t(col * K::kRow), r_base = stage + uint32_t(K::kBytes + col * KR::kRow);
      asm volatile("" : "+v"(k_base), "+v"(r_base));
      v16f s[2] = {v16f{}, v16f{}};
#pragma unroll
      for (int k = 0; k < DN / 16; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) {  // keys 32 t ..: their swizzle is that of row `col`
          const lds_char* const p = reinterpret_cast<const lds_char*>(uintptr_t(k_base + ((uint32_t(2 * k + h) ^ k_key) << 4))) + t * 32 * K::kRow;
          s[t] = mfma<kBf16>(__builtin_bit_cast(uint4, *reinterpret_cast<const lds_u32x4*>(p)), q[k], s[t]);
        }
#pragma unroll
      for (int k = 0; k < R / 16; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const lds_char* const p = reinterpret_cast<const lds_char*>(uintptr_t(r_base + ((uint32_t(2 * k + h) ^ r_key) << 4))) + t * 32 * KR::kRow;
          s[t] = mfma<kBf16>(__builtin_bit_cast(uint4, *reinterpret_cast<const lds_u32x4*>(p)), q[DN / 16 + k], s[t]);
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = s[t][e] * a.scale_log2;
      if (key0 + kKeys > wave_lo) {  // uniform
        const int seen = mine - key0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[t][e] = 32 * t + 8 * (e >> 2) + 4 * h + (e & 3) < seen ? x[t][e] : -INFINITY;
      }
      float top = x[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[t][e]);
      return max_halves(top);
    };
    // Raises the running maximum where a score is far above it.
    const auto raise = [&](float top) __attribute__((always_inline)) {
      if (__ballot(top > m_run + kLazy) == 0) return;  // uniform, and mostly so after the first block
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_new == m_run ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
      m_run = m_new;
    };
    if (wild && !idle) {
      // Which weights of this lane's query are not 0: bit 16 t + e of its half's word is key 32 t + 8 (e / 4) +
      // 4 half + e % 4.  A weight of 0 makes NaN of an infinity, as it does in the products.
      float x[2][16];
      raise(score(x));
      const float use = m_run == -INFINITY ? 0.0f : m_run;
      uint32_t some = 0u;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float* const y = &x[e >> 3][2 * (e & 7)];
        const uint32_t p = pack2<kBf16>(__builtin_amdgcn_exp2f(y[0] - use), __builtin_amdgcn_exp2f(y[1] - use));
        some |= (uint32_t((p & 0xFFFFu) != 0u) | uint32_t(p >> 16 != 0u) << 1) << (2 * e);
      }
      const auto halves = __builtin_amdgcn_permlane32_swap(some, some, false, false);
#pragma unroll 1
      for (int r = late; r < end; ++r) {
        if (key0 + r >= mine) break;
        const uint32_t bit = uint32_t(r >> 5 << 4 | (r >> 3 & 3) << 2 | (r & 3)), weighs = (r >> 2 & 1 ? halves[1] : halves[0]) >> bit & 1u;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // columns 32 d + 8 e + 4 h ..: half h of chunk 4 d + e
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            const u32x2 v = *reinterpret_cast<const __attribute__((address_space(3))) u32x2*>(
                uintptr_t(v_stage + uint32_t(r * V::kRow + (((4 * d + e) ^ V::key(r)) << 4) + 8 * h)));
#pragma unroll
            for (int f = 0; f < 4; ++f)
              if (wild_halves<kBf16>(v[f >> 1]) >> (f & 1) & 1u) o[d][4 * e + f] += weighs ? half_value<kBf16>(v[f >> 1], f & 1) : NAN;
            __builtin_amdgcn_sched_barrier(0);  // one load at a time: registers are short
          }
      }
    }
    if (wild) clean();
    if (idle) continue;

    float x[2][16];
    raise(score(x));
    const float use = m_run == -INFINITY ? 0.0f : m_run;
    // P rounded to the values' type, and summed as rounded: numerator and denominator hold the same weights.
    uint32_t p[16];
    const uint32_t ones = kBf16 ? 0x3F803F80u : 0x3C003C00u;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float* const y = &x[e >> 3][2 * (e & 7)];
      p[e] = pack2<kBf16>(__builtin_amdgcn_exp2f(y[0] - use), __builtin_amdgcn_exp2f(y[1] - use));
      l_run = dot2_ones<kBf16>(p[e], l_run, ones);
    }
    uint32_t v_base = v_stage + uint32_t(v_row * V::kRow + 8 * (j16 & 1));
    asm volatile("" : "+v"(v_base));
#pragma unroll
    for (int t = 0; t < 4; ++t) {  // keys 16 t ..: registers 8 t .. of S^T
      const uint4 w = make_uint4(p[4 * t], p[4 * t + 1], p[4 * t + 2], p[4 * t + 3]);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        uint2 v[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t c = uint32_t(4 * d + v_chunk) ^ uint32_t(V::key(v_row + 8 * g));
          lds_char* const at = reinterpret_cast<lds_char*>(uintptr_t(v_base + (c << 4))) + (16 * t + 8 * g) * V::kRow;
          v[g] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(at)));
        }
        o[d] = mfma<kBf16>(make_uint4(v[0].x, v[0].y, v[1].x, v[1].y), w, o[d]);
      }
    }
  }
  const float l = sum_halves(l_run);
  if (row >= nq) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t out = (int64_t(q0 + row) * a.n_heads + head) * DV + 4 * h;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) y[f] = o[d][4 * e + f] * inv;
      const int64_t at = out + 32 * d + 8 * e;
      if (a.out_dtype == IT_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
      else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = make_uint2(pack2<kBf16>(y[0], y[1]), pack2<kBf16>(y[2], y[3]));
    }
}

template <bool kBf16, int DN, int R, int DV>
hipError_t launch(const LatentPrefillArgs& a, hipStream_t s) {
  static std::atomic<uint64_t> opted{0};
  constexpr int lds = 2 * kKeys * (DN + R + DV) * 2;
  auto* const kern = latent_prefill<kBf16, DN, R, DV>;
  if (const hipError_t e = opt_in_lds(reinterpret_cast<const void*>(kern), lds, opted); e != hipSuccess) return e;
  const int n_qb = (a.max_q_len + kQueries - 1) / kQueries;
  const int64_t wgs = (int64_t(a.n_seqs) * a.n_heads + 7) / 8 * 8 * n_qb;
  hipLaunchKernelGGL(kern, dim3(unsigned(wgs)), dim3(kThreads), lds, s, a, n_qb);
  return hipGetLastError();
}
template <bool kBf16>
bool launch_widths(const LatentPrefillArgs& a, hipStream_t s, hipError_t& e) {
  if (a.nope == 128 && a.v_dim == 128 && a.rope == 64) e = launch<kBf16, 128, 64, 128>(a, s);
  else if (a.nope == 128 && a.v_dim == 128 && a.rope == 32) e = launch<kBf16, 128, 32, 128>(a, s);
  else if (a.nope == 128 && a.v_dim == 64 && a.rope == 64) e = launch<kBf16, 128, 64, 64>(a, s);
  else if (a.nope == 128 && a.v_dim == 64 && a.rope == 32) e = launch<kBf16, 128, 32, 64>(a, s);
  else if (a.nope == 64 && a.v_dim == 64 && a.rope == 64) e = launch<kBf16, 64, 64, 64>(a, s);
  else if (a.nope == 64 && a.v_dim == 64 && a.rope == 32) e = launch<kBf16, 64, 32, 64>(a, s);
  else return false;
  return true;
}
}  // namespace

namespace itkv {
bool latent_prefill_matrix(const LatentPrefillArgs& a, int32_t dtype, hipStream_t s, hipError_t& e) {
  if (dtype != IT_F16 && dtype != IT_BF16) return false;
  // Whole 16-byte chunks from aligned rows, and 64 rows within a 32-bit offset.
  const auto whole = [](const void* p, int64_t token, int64_t head) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && token % 8 == 0 && head % 8 == 0 && token < int64_t(1) << 24;
  };
  if (!whole(a.k, a.k_stride, a.k_head) || !whole(a.v, a.v_stride, a.v_head) || !whole(a.k_rope, a.rope_stride, 0)) return false;
  const int64_t n_qb = (a.max_q_len + kQueries - 1) / kQueries;
  if ((int64_t(a.n_seqs) * a.n_heads + 7) / 8 * 8 * n_qb > int64_t(1) << 30) return false;
  return dtype == IT_BF16 ? launch_widths<true>(a, s, e) : launch_widths<false>(a, s, e);
}
}  // namespace itkv
