// it_latent.hip -- latent rows into the cache: the latent part normalised, the
// shared rope key turned to its position, and the rope part of the query heads
// beside them.
//
//   c' = c * rsqrt(mean(c^2) + eps) * w,  r' = R(p) r,  q' = R(p) q
//
// Bound by memory, and by latency for single tokens: each row is read and
// written once, whole 16-byte vectors per lane.  A wave takes one token's row
// (its sum of squares is a sum over the wave's lanes, no LDS), the rope part of a run
// of its heads, or both; it computes the token's angles for itself, a pair per lane, as
// the rotation of K and V rows does.
// 4001 tokens of 512 + 64 elements and 32 heads in f16, rows handed back: 11.3 us, 47 MB
// (7.0 us at a copy's rate; 15.0 before positions and angles were loaded beside the rows
// and stores were converted without a branch).  One token of 28 heads: 3.0 us, latency.
#include <hip/hip_runtime.h>

#include "it_latent.hpp"
#include "it_rotary.hpp"
#include "it_strided.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kHeadSteps = 2;  // rows of heads that a lane takes

struct LatentAppendArgs {
  const char* kv;
  const char* q;
  const void* weight;
  char* pool;
  char* q_out;
  char* rows_out;
  const int64_t* slots;
  const int32_t* positions;
  const double* turns;  // NULL: nothing turns
  uint32_t* err;
  int64_t kv_stride, q_stride, q_head, out_stride, out_head, n_slots;
  float eps, magnitude;
  int n_tokens, n_heads, latent, rope, layout, cache_dtype, weight_dtype, out_dtype;
  int parts;  // waves of a token: its row's, then its heads'
  int apart;  // 1: the row has a wave of its own
  RowSplit split;
};

__device__ __forceinline__ char* row_of(const LatentAppendArgs& a, int64_t slot) {
  return a.pool + slot * int64_t(a.latent + a.rope) * (a.cache_dtype == IT_F32 ? 4 : 2);
}

template <int V>
__device__ __forceinline__ void load_weight(const LatentAppendArgs& a, int e, float (&w)[V]) {
  if (a.weight_dtype == IT_F32)
    RowVec<IT_F32, V>::widen(*reinterpret_cast<const typename RowVec<IT_F32, V>::raw*>(static_cast<const float*>(a.weight) + e), w);
  else if (a.weight_dtype == IT_BF16)
    RowVec<IT_BF16, V>::widen(*reinterpret_cast<const typename RowVec<IT_BF16, V>::raw*>(static_cast<const uint16_t*>(a.weight) + e), w);
  else
    RowVec<IT_F16, V>::widen(*reinterpret_cast<const typename RowVec<IT_F16, V>::raw*>(static_cast<const uint16_t*>(a.weight) + e), w);
}

// Whether a token is written at all (false: a bad position), and its slot, -1 where it is not one.
__device__ __forceinline__ bool token_ok(const LatentAppendArgs& a, bool latch, int pos, int64_t& slot) {
  if (pos < 0) {
    if (latch) atomicOr(a.err, kErrPos);
    return false;
  }
  if (slot >= a.n_slots) {
    if (latch) atomicOr(a.err, kErrSlot);
    slot = -1;
  }
  return true;
}

// V elements to `dtype`, which is SRC where kSame: chosen when the kernel was, and converted
// without a branch (its own NaN for fp16's).
template <int SRC, bool kSame, int V>
__device__ __forceinline__ void put_vec(void* base, int64_t element, int dtype, const float (&x)[V]) {
  if constexpr (kSame && SRC == IT_F16) {
    typedef uint32_t words __attribute__((ext_vector_type(V / 2)));
    words w;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = f32_to_f16_bits(x[2 * i]) | f32_to_f16_bits(x[2 * i + 1]) << 16;
    *reinterpret_cast<words*>(static_cast<uint16_t*>(base) + element) = w;
  } else {
    store_row_vec<V>(base, element, kSame ? SRC : dtype, x);
  }
}

// Vectors of V elements of SRC (16 bytes), aligned.  kSame: the cache's and q_out's type is SRC.
template <int SRC, bool kSame>
__global__ __launch_bounds__(kThreads) void latent_append_rows(LatentAppendArgs a) {
  constexpr int es = SRC == IT_F32 ? 4 : 2, V = 16 / es;
  constexpr int kMaxVecs = 1024 / (64 * V);  // a lane's vectors of a latent
  constexpr int kMaxTurns = 2;               // and pairs of a rope part: 256 elements
  using In = RowVec<SRC, V>;
  extern __shared__ __attribute__((aligned(16))) float2 angles[];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = int(threadIdx.x & 63);
  const int task = int(blockIdx.x) * kWaves + wave, t = task / a.parts, part = task - t * a.parts;
  if (t >= a.n_tokens) return;  // uniform
  // The token's row is its first wave's; the heads begin with that or with the next.
  const bool with_row = part == 0;
  const int head_part = part - a.apart;
  const RowSplit& s = a.split;
  float2* const own = angles + wave * angle_room<V>(a.rope);
  const int sub = int((uint32_t(lane) * s.inv) >> 16), c = lane - sub * s.lanes;
  const int h0 = head_part * (s.rows * kHeadSteps) + sub;
  LanePairs<V> lp(s, c);
  // All loads before the first of what follows from the token's position.
  const int pos = a.turns ? a.positions[t] : 0;
  int64_t slot = a.slots[t];
  double turns[kMaxTurns];
  if (a.turns) {
#pragma unroll
    for (int j = 0; j < kMaxTurns; ++j)
      if (j * 128 < a.rope) turns[j] = a.turns[min(j * 64 + lane, (a.rope >> 1) - 1)];
  }
  typename In::raw xa[kHeadSteps], xb[kHeadSteps];
  const bool heads = head_part >= 0 && a.n_heads > 0;  // uniform
  if (heads) {
#pragma unroll
    for (int j = 0; j < kHeadSteps; ++j) {  // past the last head a lane reads it again; only the stores are predicated
      const int h = min(h0 + j * s.rows, a.n_heads - 1);
      const char* const src = a.q + (t * a.q_stride + h * a.q_head) * es;
      xa[j] = *reinterpret_cast<const typename In::raw*>(src + lp.ea * es);
      xb[j] = *reinterpret_cast<const typename In::raw*>(src + lp.eb * es);
    }
  }
  const char* const src = a.kv + t * a.kv_stride * es;
  const int vecs = a.latent / V;
  const bool turner = lane < s.lanes;
  typename In::raw x[kMaxVecs], ra, rb;
  float weight[V];
  if (with_row) {
#pragma unroll
    for (int j = 0; j < kMaxVecs; ++j)
      if (j * 64 < vecs) x[j] = *reinterpret_cast<const typename In::raw*>(src + min(j * 64 + lane, vecs - 1) * 16);
    if (turner) {
      ra = *reinterpret_cast<const typename In::raw*>(src + (a.latent + lp.ea) * es);
      rb = *reinterpret_cast<const typename In::raw*>(src + (a.latent + lp.eb) * es);
    }
    if (a.weight) load_weight(a, min(lane, vecs - 1) * V, weight);  // the first vector's
  }
  if (!token_ok(a, with_row && lane == 0, pos, slot)) return;  // uniform
  if (a.turns) {
#pragma unroll
    for (int j = 0; j < kMaxTurns; ++j) {
      if (j * 128 >= a.rope) continue;  // uniform
      const float2 cs = rotary_angle(turns[j], pos);
      if (j * 128 + 2 * lane < a.rope) own[j * 64 + lane] = make_float2(cs.x * a.magnitude, cs.y * a.magnitude);
    }
    wave_lds_fence();
    lp.load(s, own);
  }
  if (heads) {
#pragma unroll
    for (int j = 0; j < kHeadSteps; ++j) {
      const int h = h0 + j * s.rows;
      if (h >= a.n_heads || sub >= s.rows) continue;
      float fa[V], fb[V];
      In::widen(xa[j], fa);
      In::widen(xb[j], fb);
      if (a.turns) lp.turn(s, fa, fb);
      const int64_t at = t * a.out_stride + h * a.out_head;
      put_vec<SRC, kSame, V>(a.q_out, at + lp.ea, a.out_dtype, fa);
      put_vec<SRC, kSame, V>(a.q_out, at + lp.eb, a.out_dtype, fb);
    }
  }
  if (!with_row) return;  // uniform
  float norm = 1.0f;
  if (a.weight) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxVecs; ++j) {
      if (j * 64 + lane >= vecs) continue;
      float f[V];
      In::widen(x[j], f);
#pragma unroll
      for (int e = 0; e < V; ++e) sum = fmaf(f[e], f[e], sum);
    }
    norm = 1.0f / sqrtf(group_sum<64>(sum) / float(a.latent) + a.eps);
  }
  const int64_t row = int64_t(a.latent + a.rope);
  char* const to = slot >= 0 ? row_of(a, slot) : nullptr;
  const auto put = [&](int e, const float(&f)[V]) {
    if (to) put_vec<SRC, kSame, V>(to, e, a.cache_dtype, f);
    if (a.rows_out) put_vec<SRC, kSame, V>(a.rows_out, t * row + e, a.cache_dtype, f);
  };
#pragma unroll
  for (int j = 0; j < kMaxVecs; ++j) {
    const int v = j * 64 + lane;
    if (v >= vecs) continue;
    float f[V];
    In::widen(x[j], f);
    if (a.weight) {
      if (j > 0) load_weight(a, v * V, weight);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = f[e] * norm * weight[e];
    }
    put(v * V, f);
  }
  if (turner) {
    float fa[V], fb[V];
    In::widen(ra, fa);
    In::widen(rb, fb);
    if (a.turns) lp.turn(s, fa, fb);
    put(a.latent + lp.ea, fa);
    put(a.latent + lp.eb, fb);
  }
}

// The same, element by element: rows that are not aligned to vectors, or whose
// pairs do not fall into them.
template <int SRC>
__global__ __launch_bounds__(kThreads) void latent_append_general(LatentAppendArgs a) {
  constexpr int es = SRC == IT_F32 ? 4 : 2;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = int(threadIdx.x & 63);
  const int task = int(blockIdx.x) * kWaves + wave, t = task / a.parts, part = task - t * a.parts;
  if (t >= a.n_tokens) return;
  const int pos = a.turns ? a.positions[t] : 0;
  int64_t slot = a.slots[t];
  if (!token_ok(a, part == 0 && lane == 0, pos, slot)) return;
  const int half = a.rope >> 1, es_out = a.out_dtype == IT_F32 ? 4 : 2;
  const bool halves = a.layout == IT_ROTARY_HALF;
  const int64_t row = int64_t(a.latent + a.rope);
  char* const to = slot >= 0 ? row_of(a, slot) : nullptr;
  // A lane per pair of a head (or of the row): it reads both elements before it writes them.
  const auto pair = [&](const char* from, int p, auto&& put) {
    const int e0 = halves ? p : 2 * p, e1 = halves ? p + half : 2 * p + 1;
    float x = load_element(from, e0, SRC), y = load_element(from, e1, SRC);
    if (a.turns) {
      float2 cs = rotary_angle(a.turns[p], pos);
      cs = make_float2(cs.x * a.magnitude, cs.y * a.magnitude);
      LanePairs<4>::pair(cs, x, y);
    }
    put(e0, x);
    put(e1, y);
  };
  if (part > 0) {
    const int heads = min(a.n_heads - (part - 1) * a.split.rows, a.split.rows);
    for (int i = lane; i < heads * half; i += 64) {
      const int h = (part - 1) * a.split.rows + i / half;
      char* const out = a.q_out + (t * a.out_stride + h * a.out_head) * es_out;
      pair(a.q + (t * a.q_stride + h * a.q_head) * es, i % half, [&](int e, float f) { store_element(out, e, a.out_dtype, f); });
    }
    return;
  }
  const char* const src = a.kv + t * a.kv_stride * es;
  const auto put = [&](int e, float f) {
    if (to) store_element(to, e, a.cache_dtype, f);
    if (a.rows_out) store_element(a.rows_out, t * row + e, a.cache_dtype, f);
  };
  float norm = 1.0f;
  if (a.weight) {
    float sum = 0.0f;
    for (int e = lane; e < a.latent; e += 64) {
      const float f = load_element(src, e, SRC);
      sum = fmaf(f, f, sum);
    }
    norm = 1.0f / sqrtf(group_sum<64>(sum) / float(a.latent) + a.eps);
  }
  for (int e = lane; e < a.latent; e += 64) {
    const float f = load_element(src, e, SRC);
    put(e, a.weight ? f * norm * load_element(a.weight, e, a.weight_dtype) : f);
  }
  for (int p = lane; p < half; p += 64) pair(src + a.latent * es, p, [&](int e, float f) { put(a.latent + e, f); });
}

inline bool is_float(int32_t dt) { return dt == IT_F32 || dt == IT_F16 || dt == IT_BF16; }
inline bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(to) == 0; }
}  // namespace

extern "C" int32_t it_latent_append(it_kv_cache* c, const it_rotary* rotary, const void* kv, int32_t src_dtype, int64_t kv_stride,
                                    const void* weight, int32_t weight_dtype, float eps, const void* q, int64_t q_stride,
                                    int64_t q_head_stride, int32_t n_heads, void* q_out, int32_t q_out_dtype, int64_t out_stride,
                                    int64_t out_head_stride, void* rows_out, const int64_t* slot_mapping, const int32_t* positions,
                                    int32_t n_tokens, void* stream) {
  const char* who = "it_latent_append";
  if (!c) return fail(IT_INVALID_INPUT, "%s: cache is NULL", who);
  if (!c->latent_dim) return fail(IT_INVALID_INPUT, "%s: not a latent cache", who);
  if (int32_t rc = one_layer(c, who)) return rc;
  if (!is_float(src_dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: src_dtype %d (F32, F16 or BF16)", who, src_dtype);
  if (weight && !is_float(weight_dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: weight dtype %d (F32, F16 or BF16)", who, weight_dtype);
  if (weight && !(eps >= 0.0f && eps < INFINITY)) return fail(IT_INVALID_INPUT, "%s: eps %g", who, double(eps));
  if (n_tokens < 0 || n_heads < 0 || n_heads > 65536) return fail(IT_INVALID_INPUT, "%s: n_tokens %d, n_heads %d", who, n_tokens, n_heads);
  if (n_heads && !is_float(q_out_dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: q_out dtype %d (F32, F16 or BF16)", who, q_out_dtype);
  const int latent = c->latent_dim, rope = c->head_dim - latent;
  if (rotary && rotary->n_dims != rope)
    return fail(IT_INVALID_INPUT, "%s: %d rotated elements, the cache's rope part has %d", who, rotary->n_dims, rope);
  if (rotary && rotary->device != c->device) return fail(IT_INVALID_INPUT, "%s: rotary and cache on different devices", who);
  const int64_t row = c->head_dim, es = dtype_bytes(src_dtype), os = n_heads ? dtype_bytes(q_out_dtype) : 4, kFar = int64_t(1) << 40;
  if (n_tokens <= 1) kv_stride = row, q_stride = out_stride = 0;  // not used
  if (n_heads <= 1) q_head_stride = out_head_stride = 0;
  if (n_tokens > 1 && (kv_stride < row || kv_stride > kFar))
    return fail(IT_INVALID_INPUT, "%s: kv_stride %lld below a row's %lld elements (or above 2^40)", who, (long long)kv_stride, (long long)row);
  // Neither a token's heads nor the tokens of a head may lie in one another.
  const auto fits = [&](int64_t token, int64_t head) {
    if (token < 0 || head < 0 || token > kFar || head > kFar) return false;
    if (n_heads > 1 && head < rope) return false;
    if (n_tokens > 1 && token < rope) return false;
    return n_heads <= 1 || n_tokens <= 1 || token >= head * (n_heads - 1) + rope || head >= token * (n_tokens - 1) + rope;
  };
  if (n_heads && (!fits(q_stride, q_head_stride) || !fits(out_stride, out_head_stride)))
    return fail(IT_INVALID_INPUT, "%s: q strides %lld, %lld and q_out strides %lld, %lld do not hold rows of %d elements apart", who,
                (long long)q_stride, (long long)q_head_stride, (long long)out_stride, (long long)out_head_stride, rope);
  if (n_tokens == 0) return IT_OK;
  if (!kv || !slot_mapping || (rotary && !positions) || (n_heads && (!q || !q_out))) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  if (!aligned(kv, es) || (weight && !aligned(weight, dtype_bytes(weight_dtype))) || (n_heads && (!aligned(q, es) || !aligned(q_out, os))) ||
      (rows_out && !aligned(rows_out, dtype_bytes(c->dtype))))
    return fail(IT_INVALID_INPUT, "%s: tensors must be aligned to their elements", who);
  // What is written may lie between the rows of what is read (parts of one projection), not on them.
  const int64_t cs = dtype_bytes(c->dtype);
  const auto rows_at = [](const void* p, int64_t token, int64_t head, int64_t elements, int64_t size, int64_t tokens, int64_t heads) {
    return StridedRows{reinterpret_cast<uintptr_t>(p), token * size, head * size, elements * size, tokens, heads};
  };
  const StridedRows r_kv = rows_at(kv, kv_stride, 0, row, es, n_tokens, 1), r_rows = rows_at(rows_out, row, 0, row, cs, n_tokens, 1);
  if (n_heads) {
    const StridedRows r_q = rows_at(q, q_stride, q_head_stride, rope, es, n_tokens, n_heads);
    const StridedRows r_out = rows_at(q_out, out_stride, out_head_stride, rope, os, n_tokens, n_heads);
    const bool same = q == q_out && src_dtype == q_out_dtype && q_stride == out_stride && q_head_stride == out_head_stride;
    if ((!same && share_memory(r_out, r_q)) || share_memory(r_out, r_kv))
      return fail(IT_INVALID_INPUT, "%s: q_out overlaps q or kv (it may be q itself, with its strides and dtype)", who);
    if (rows_out && share_memory(r_out, r_rows)) return fail(IT_INVALID_INPUT, "%s: q_out overlaps rows_out", who);
    if (rows_out && share_memory(r_q, r_rows)) return fail(IT_INVALID_INPUT, "%s: rows_out overlaps q", who);
  }
  if (rows_out && share_memory(r_kv, r_rows)) return fail(IT_INVALID_INPUT, "%s: rows_out overlaps kv", who);
  LatentAppendArgs a{};
  a.kv = static_cast<const char*>(kv);
  a.q = static_cast<const char*>(n_heads ? q : nullptr);
  a.weight = weight;
  a.pool = static_cast<char*>(c->k_pool);
  a.q_out = static_cast<char*>(n_heads ? q_out : nullptr);
  a.rows_out = static_cast<char*>(rows_out);
  a.slots = slot_mapping;
  a.positions = positions;
  a.turns = rotary ? rotary->turns : nullptr;
  a.err = c->err_flag;
  a.kv_stride = kv_stride;
  a.q_stride = q_stride;
  a.q_head = q_head_stride;
  a.out_stride = out_stride;
  a.out_head = out_head_stride;
  a.n_slots = c->num_blocks * c->block_size;
  a.eps = eps;
  a.magnitude = rotary ? rotary->magnitude : 1.0f;
  a.n_tokens = n_tokens;
  a.n_heads = n_heads;
  a.latent = latent;
  a.rope = rope;
  a.layout = rotary ? rotary->layout : IT_ROTARY_INTERLEAVED;
  a.cache_dtype = c->dtype;
  a.weight_dtype = weight ? weight_dtype : IT_F32;
  a.out_dtype = n_heads ? q_out_dtype : IT_F32;
  // Vectors: 16 bytes of the source's type, stored as as many elements of the
  // cache's and q_out's types (their alignment: that many elements', 16 bytes at most).
  const int v = src_dtype == IT_F32 ? 4 : 8;
  const auto vec = [&](const void* p, int64_t s0, int64_t s1, int64_t e) {
    const int64_t to = v * e < 16 ? v * e : 16;
    return aligned(p, to) && s0 * e % to == 0 && s1 * e % to == 0;
  };
  const bool fast = row_split(rope, rope, a.layout, v, v, a.split) && vec(kv, kv_stride, 0, es) &&
                    (!weight || vec(weight, 0, 0, dtype_bytes(weight_dtype))) &&
                    (!n_heads || (vec(q, q_stride, q_head_stride, es) && vec(q_out, out_stride, out_head_stride, os))) &&
                    (!rows_out || vec(rows_out, 0, 0, dtype_bytes(c->dtype)));
  if (!fast) {
    a.split.rows = 16;  // heads of a wave in the general kernel
    a.parts = 1 + (n_heads + 15) / 16;
  } else {
    // The row has a wave of its own (one token of 28 heads 3.0 us against 3.7 where the row and the
    // first heads share one, 600 of 128 6.6 against 7.2, 4001 of 32 11.3 against 11.6), unless there
    // are few heads and more tokens than waves are resident: then the angles cost more (8191 of 4
    // 13.6 against 12.1).
    const int head_waves = (n_heads + a.split.rows * kHeadSteps - 1) / (a.split.rows * kHeadSteps);
    a.apart = head_waves > 0 && (n_heads * 4 > a.split.rows * kHeadSteps || int64_t(n_tokens) * 2 <= 256 * 32);
    a.parts = a.apart + (head_waves > 1 ? head_waves : 1);
  }
  if (int64_t(n_tokens) * a.parts > int64_t(1) << 30) return fail(IT_INVALID_INPUT, "%s: %d tokens of %d heads", who, n_tokens, n_heads);
  int dev = -1;
  (void)hipGetDevice(&dev);
  if (dev != c->device) (void)hipSetDevice(c->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(unsigned((n_tokens * a.parts + kWaves - 1) / kWaves));
  const size_t lds = size_t(kWaves) * (v == 4 ? angle_room<4>(rope) : angle_room<8>(rope)) * sizeof(float2);
  const bool same = c->dtype == src_dtype && (!n_heads || q_out_dtype == src_dtype);
  const auto launch = [&](auto* kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), fast ? lds : 0, s, a); };
  switch (src_dtype) {
    case IT_F32: launch(!fast ? latent_append_general<IT_F32> : same ? latent_append_rows<IT_F32, true> : latent_append_rows<IT_F32, false>); break;
    case IT_BF16: launch(!fast ? latent_append_general<IT_BF16> : same ? latent_append_rows<IT_BF16, true> : latent_append_rows<IT_BF16, false>); break;
    default: launch(!fast ? latent_append_general<IT_F16> : same ? latent_append_rows<IT_F16, true> : latent_append_rows<IT_F16, false>); break;
  }
  const hipError_t e = hipGetLastError();
  if (dev >= 0 && dev != c->device) (void)hipSetDevice(dev);
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
