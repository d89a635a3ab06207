// it_latent_attn.hip -- latent attention: the C ABI of its absorbed and expanded
// forms, and the kernels for every type and width, in fp32 on the vector units.
// 16-bit rows of the usual widths run on the matrix cores instead
// (it_latent_decode.hpp, it_latent_prefill.hip).  A query row a workgroup, so that every
// head reads a sequence's rows again: F32 rows of 512 + 64 elements, 32 sequences of 256 to
// 8192 tokens, 32 heads, 15.9 ms; prompt chunks of 512 over 1536 to 2560 keys, 8 x 32 heads,
// 116 ms.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "it_latent.hpp"
#include "it_rows.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxWidth = 1280;            // a key's elements: 1024 + 256
constexpr int kKeyRegs = kMaxWidth / 64;   // of them a lane's
constexpr int kMaxValue = 1024;
constexpr int kValueRegs = kMaxValue / 64;

// One query row against keys [lo, hi): a workgroup, each wave every fourth key,
// with a running maximum and sum of its own; the four are joined in LDS.  A lane
// holds elements lane, lane + 64, .. of the query and of the result, and a key's
// score is a sum over the wave.  Bound by that sum's latency, key after key.
//   key(j, e): element e of key j, value(j, e) of its value
template <class Query, class Key, class Value>
__device__ __forceinline__ void attend_row(int width, int v_dim, int lo, int hi, float scale_log2, Query&& query, Key&& key,
                                           Value&& value, void* out, int64_t at, int out_dtype) {
  __shared__ float part[kWaves][kMaxValue];
  __shared__ float2 ml[kWaves];
  const int lane = int(threadIdx.x & 63), wave = int(threadIdx.x >> 6);
  float q[kKeyRegs], o[kValueRegs], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kKeyRegs; ++i) q[i] = i * 64 + lane < width ? query(i * 64 + lane) : 0.0f;
#pragma unroll
  for (int i = 0; i < kValueRegs; ++i) o[i] = 0.0f;
  for (int j = lo + wave; j < hi; j += kWaves) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kKeyRegs; ++i)
      if (i * 64 + lane < width) s = fmaf(q[i], key(j, i * 64 + lane), s);
    s = group_sum<64>(s) * scale_log2;
    const float m_new = fmaxf(m, s);  // a NaN score leaves it, and makes the sum NaN
    const float use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = exp2f(m - use), p = exp2f(s - use);
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < kValueRegs; ++i)
      if (i * 64 + lane < v_dim) o[i] = fmaf(p, value(j, i * 64 + lane), o[i] * alpha);
    m = m_new;
  }
  if (lane == 0) ml[wave] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < kValueRegs; ++i)
    if (i * 64 + lane < v_dim) part[wave][i * 64 + lane] = o[i];
  __syncthreads();
  float M = ml[0].x, L = 0.0f, w[kWaves];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    w[i] = ml[i].x == -INFINITY && ml[i].y == 0.0f ? 0.0f : exp2f(ml[i].x - M);
    L = fmaf(w[i], ml[i].y, L);
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // no key seen: 0
  for (int e = int(threadIdx.x); e < v_dim; e += kThreads) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      if (w[i] != 0.0f) x = fmaf(w[i], part[i][e], x);
    store_element(out, at + e, out_dtype, x * inv);
  }
}

// grid: (row of the sequence, sequence).
template <int DT>
__global__ __launch_bounds__(kThreads) void latent_decode_general(LatentDecodeArgs a) {
  const int b = int(blockIdx.y), r = int(blockIdx.x), i = r / a.n_heads, h = r - i * a.n_heads;
  const LatentSpan span = latent_span(a, b, r == 0 && threadIdx.x == 0);
  const int hi = min(span.ctx, max(span.ctx - a.q_len + 1 + i, span.start));
  const int64_t t = int64_t(b) * a.q_len + i;
  const int bs = 1 << a.log2_bs, row = a.latent + a.rope;
  const int32_t* const bt = a.bt + int64_t(b) * a.max_blocks;
  // A block id outside the pool is latched and its keys are read from block 0.
  const auto at = [&](int j, int e) {
    int64_t blk = bt[j >> a.log2_bs];
    if (blk < 0 || blk >= a.num_blocks) {
      if ((threadIdx.x & 63) == 0) atomicOr(a.err, kErrBlock);
      blk = 0;
    }
    return load_element(a.pool + blk * a.page_bytes, int64_t(j & (bs - 1)) * row + e, DT);
  };
  attend_row(
      row, a.latent, span.start, hi, a.scale_log2,
      [&](int e) {
        return e < a.latent ? load_element(a.q_latent, t * a.ql_stride + h * a.ql_head + e, DT)
                            : load_element(a.q_rope, t * a.qr_stride + h * a.qr_head + e - a.latent, DT);
      },
      at, at, a.out, (t * a.n_heads + h) * a.latent, a.out_dtype);
}

// grid: (query of the sequence, head, sequence).
template <int DT>
__global__ __launch_bounds__(kThreads) void latent_prefill_general(LatentPrefillArgs a) {
  const int b = int(blockIdx.z), h = int(blockIdx.y), i = int(blockIdx.x);
  const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  if (!latent_prefill_fits(a, q0, q1, k0, k1) || i >= q1 - q0) return;
  const int n = k1 - k0, hi = a.causal ? max(0, n - (q1 - q0) + i + 1) : n;
  const int64_t t = q0 + i;
  attend_row(
      a.nope + a.rope, a.v_dim, 0, hi, a.scale_log2, [&](int e) { return load_element(a.q, t * a.q_stride + h * a.q_head + e, DT); },
      [&](int j, int e) {
        return e < a.nope ? load_element(a.k, (k0 + j) * a.k_stride + h * a.k_head + e, DT)
                          : load_element(a.k_rope, (k0 + j) * a.rope_stride + e - a.nope, DT);
      },
      [&](int j, int e) { return load_element(a.v, (k0 + j) * a.v_stride + h * a.v_head + e, DT); }, a.out,
      (t * a.n_heads + h) * a.v_dim, a.out_dtype);
}

inline bool is_float(int32_t dt) { return dt == IT_F32 || dt == IT_F16 || dt == IT_BF16; }
inline bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(to) == 0; }
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int64_t kFar = int64_t(1) << 40;

int32_t decode_sizes(const char* who, const it_kv_cache* c, int32_t n_seqs, int32_t q_len, int32_t n_heads, int32_t max_tokens) {
  if (!c) return fail(IT_INVALID_INPUT, "%s: cache is NULL", who);
  if (!c->latent_dim) return fail(IT_INVALID_INPUT, "%s: not a latent cache", who);
  if (n_seqs < 0 || n_seqs > 65535 || q_len < 1 || q_len > kLatentMaxQ || n_heads < 1 || n_heads > 1024 || max_tokens < 0)
    return fail(IT_INVALID_INPUT, "%s: n_seqs %d (to 65535), q_len %d (1 to %d), n_heads %d (1 to 1024), max_tokens %d", who, n_seqs,
                q_len, kLatentMaxQ, n_heads, max_tokens);
  return IT_OK;
}
}  // namespace

namespace {
constexpr int kTile = 32;  // of the matrix-core kernels: cached tokens
// Query groups and token groups of a workgroup, by the call's groups of 16 queries and the
// tiles that a CU gets of it (by max_tokens).  Many query groups read a tile from LDS and from
// memory once for all; few have partial results that are as much smaller, and more waves on a
// piece's own latency.
//   Rows of up to 288 elements, of which LDS holds two tiles for each of four token groups: two
// query groups or, of one and below 6 tiles, one (L = 256, 64 heads, 16 x 12288 tokens: two
// 32 us, four with one token group 42, eight 51; 128 heads 49, 64, 54; 32 heads, 16 x 1024: one
// 12.4, two 13.4; 28 heads, 24 x 4000: 22.3, 21.3).
//   Wider ones (L = 512, one, two, four and eight groups): below 10 tiles 28 heads over 1 x 1023
// tokens 15.0, 16.0, 17.6, 22.0 us, 32 over 32 x 512 18, 24, 27, 34, 64 over 16 x 2048 28, 24,
// 35, 44, 128 over 64 x 1000 67, 49, 55, 62; from there 32 over 32 x 4096 46, 40, 46, 66, 64 over
// 24 x 4096 54, 46, 43, 61, 128 over 16 x 8192 87, 85, 73, 77; from 24 on 128 over 16 x 12288
// 149, 119, 97, 96, over 16 of 8192 to 16384 the last two 123, 107.
struct HostPlan {
  int qg, workers, row_wgs;
  size_t o_bytes, ml_bytes, share_bytes;
};
HostPlan plan_of(int latent, int rope, int n_seqs, int q_len, int n_heads, int max_tokens, int n_cu) {
  HostPlan p;
  const int groups = (q_len * n_heads + 15) / 16;  // of 16 queries
  const int64_t all = int64_t(n_seqs) * ((int64_t(max_tokens) + kTile - 1) / kTile), tiles = all / n_cu;
  if (latent + rope <= kLatentNarrow) p.qg = groups == 1 || tiles < 6 ? 1 : 2;
  else if (tiles < 10) p.qg = groups <= 2 ? 1 : 2;
  else p.qg = groups <= 1 ? 1 : groups == 2 ? 2 : groups <= 4 || tiles < 24 ? 4 : 8;
  p.row_wgs = (groups + p.qg - 1) / p.qg;
  p.workers = int(std::max<int64_t>(1, std::min<int64_t>(n_cu / p.row_wgs, all + n_seqs)));
  const size_t parts = size_t(p.workers) * size_t(p.row_wgs) * 2 * size_t(p.qg);
  p.o_bytes = parts * size_t(latent) * 16 * 4;
  p.ml_bytes = parts * 16 * 8;
  p.share_bytes = size_t(n_seqs) * 8;
  return p;
}

bool takes(int32_t dtype, int latent, int rope, int block_size) {
  if ((dtype != IT_F16 && dtype != IT_BF16) || block_size < 8) return false;
  return (latent == 512 && rope == 64) || (latent == 256 && (rope == 64 || rope == 32)) || (latent == 128 && rope == 64);
}

}  // namespace

namespace itkv {
size_t latent_decode_matrix_ws(int32_t dtype, int latent, int rope, int block_size, int n_seqs, int q_len, int n_heads, int max_tokens,
                               int n_cu) {
  if (!takes(dtype, latent, rope, block_size)) return 0;
  const HostPlan p = plan_of(latent, rope, n_seqs, q_len, n_heads, max_tokens, n_cu);
  return p.o_bytes + p.ml_bytes + p.share_bytes;
}

bool latent_decode_matrix(const LatentDecodeArgs& a, int32_t dtype, int block_size, int n_cu, hipStream_t s, hipError_t& e) {
  if (!takes(dtype, a.latent, a.rope, block_size)) return false;
  const HostPlan h = plan_of(a.latent, a.rope, a.n_seqs, a.q_len, a.n_heads, a.max_tokens, n_cu);
  char* const ws = reinterpret_cast<char*>(a.ws);
  const LatentSplitPlan p{h.workers, h.row_wgs, reinterpret_cast<float4*>(ws), reinterpret_cast<float2*>(ws + h.o_bytes),
                          reinterpret_cast<int2*>(ws + h.o_bytes + h.ml_bytes)};
  e = dtype == IT_BF16 ? latent_decode_bf16(a, p, h.qg, s) : latent_decode_f16(a, p, h.qg, s);
  return true;
}

int latent_compute_units(int device) {
  static std::atomic<int> known[64];
  int n = device >= 0 && device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) return 256;
  if (device >= 0 && device < 64) known[device].store(n, std::memory_order_relaxed);
  return n;
}
}  // namespace itkv

extern "C" size_t it_latent_decode_workspace(const it_kv_cache* c, int32_t n_seqs, int32_t q_len, int32_t n_heads, int32_t max_tokens) {
  if (decode_sizes("it_latent_decode_workspace", c, n_seqs, q_len, n_heads, max_tokens)) return 0;
  return latent_decode_matrix_ws(c->dtype, c->latent_dim, c->head_dim - c->latent_dim, c->block_size, n_seqs, q_len, n_heads, max_tokens,
                                 latent_compute_units(c->device));
}

extern "C" int32_t it_latent_decode(const it_kv_cache* c, const void* q_latent, const void* q_rope, int32_t q_dtype, int64_t ql_stride,
                                    int64_t ql_head_stride, int64_t qr_stride, int64_t qr_head_stride, int32_t n_heads, int32_t q_len,
                                    const int32_t* block_tables, int32_t max_blocks, const int32_t* ctx_lens, const int32_t* start_pos,
                                    int32_t n_seqs, int32_t max_tokens, float scale, void* ws, size_t ws_bytes, void* out,
                                    int32_t out_dtype, void* stream) {
  const char* who = "it_latent_decode";
  if (int32_t rc = decode_sizes(who, c, n_seqs, q_len, n_heads, max_tokens)) return rc;
  if (int32_t rc = one_layer(c, who)) return rc;
  if (q_dtype != c->dtype) return fail(IT_NOT_IMPLEMENTED, "%s: q dtype %d, the cache's is %d", who, q_dtype, c->dtype);
  if (out_dtype != IT_F32 && out_dtype != q_dtype) return fail(IT_NOT_IMPLEMENTED, "%s: out dtype %d (F32 or q's)", who, out_dtype);
  if (max_blocks <= 0) return fail(IT_INVALID_INPUT, "%s: max_blocks %d", who, max_blocks);
  if (!(scale == scale) || std::isinf(scale)) return fail(IT_INVALID_INPUT, "%s: scale is not finite", who);
  const int64_t rows = int64_t(n_seqs) * q_len;
  if (rows <= 1) ql_stride = qr_stride = 0;  // not used
  if (n_heads == 1) ql_head_stride = qr_head_stride = 0;
  for (int64_t s : {ql_stride, ql_head_stride, qr_stride, qr_head_stride})
    if (s < 0 || s > kFar) return fail(IT_INVALID_INPUT, "%s: stride %lld", who, (long long)s);
  // All sequences' tiles are numbered in 32 bits.
  if (int64_t(n_seqs) * (std::min<int64_t>(max_tokens, int64_t(max_blocks) << c->log2_bs) / kTile + 2) > int64_t(1) << 30)
    return fail(IT_INVALID_INPUT, "%s: %d sequences of up to %d tokens: more than 2^30 runs of %d", who, n_seqs, max_tokens, kTile);
  if (n_seqs == 0) return IT_OK;
  if (!q_latent || !q_rope || !block_tables || !ctx_lens || !out) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  const int64_t es = dtype_bytes(q_dtype);
  if (!aligned(q_latent, es) || !aligned(q_rope, es) || !aligned(out, 16))
    return fail(IT_INVALID_INPUT, "%s: q must be aligned to its elements, out to 16 bytes", who);
  const size_t need = it_latent_decode_workspace(c, n_seqs, q_len, n_heads, max_tokens);
  if (need && (!ws || ws_bytes < need || !aligned(ws, 256)))
    return fail(IT_INVALID_INPUT, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", who, ws ? ws_bytes : size_t(0), need);
  LatentDecodeArgs a{};
  a.q_latent = q_latent;
  a.q_rope = q_rope;
  a.ql_stride = ql_stride;
  a.ql_head = ql_head_stride;
  a.qr_stride = qr_stride;
  a.qr_head = qr_head_stride;
  a.pool = static_cast<const char*>(c->k_pool);
  a.bt = block_tables;
  a.ctx_lens = ctx_lens;
  a.start_pos = start_pos;
  a.out = out;
  a.err = c->err_flag;
  a.ws = static_cast<float*>(ws);
  a.page_bytes = c->page_bytes;
  a.num_blocks = c->num_blocks;
  a.scale_log2 = scale * kLog2e;
  a.n_heads = n_heads;
  a.q_len = q_len;
  a.n_seqs = n_seqs;
  a.max_blocks = max_blocks;
  a.max_tokens = max_tokens;
  a.log2_bs = c->log2_bs;
  a.latent = c->latent_dim;
  a.rope = c->head_dim - c->latent_dim;
  a.out_dtype = out_dtype;
  int dev = -1;
  (void)hipGetDevice(&dev);
  if (dev != c->device) (void)hipSetDevice(c->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (!latent_decode_matrix(a, c->dtype, c->block_size, latent_compute_units(c->device), s, e)) {
    const dim3 grid(unsigned(q_len * n_heads), unsigned(n_seqs));
    switch (c->dtype) {
      case IT_F32: hipLaunchKernelGGL(latent_decode_general<IT_F32>, grid, dim3(kThreads), 0, s, a); break;
      case IT_BF16: hipLaunchKernelGGL(latent_decode_general<IT_BF16>, grid, dim3(kThreads), 0, s, a); break;
      default: hipLaunchKernelGGL(latent_decode_general<IT_F16>, grid, dim3(kThreads), 0, s, a); break;
    }
    e = hipGetLastError();
  }
  if (dev >= 0 && dev != c->device) (void)hipSetDevice(dev);
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}

extern "C" int32_t it_latent_prefill(const void* q, const void* k, const void* v, const void* k_rope, int32_t dtype, int64_t q_stride,
                                     int64_t q_head_stride, int64_t k_stride, int64_t k_head_stride, int64_t v_stride,
                                     int64_t v_head_stride, int64_t rope_stride, int32_t n_heads, int32_t nope_dim, int32_t rope_dim,
                                     int32_t v_dim, const int32_t* cu_q, const int32_t* cu_k, int32_t n_seqs, int32_t total_q,
                                     int32_t total_k, int32_t max_q_len, int32_t max_k_len, float scale, int32_t causal, void* out,
                                     int32_t out_dtype, void* stream) {
  const char* who = "it_latent_prefill";
  if (!is_float(dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: dtype %d (F32, F16 or BF16)", who, dtype);
  if (out_dtype != IT_F32 && out_dtype != dtype) return fail(IT_NOT_IMPLEMENTED, "%s: out dtype %d (F32 or q's)", who, out_dtype);
  if (n_heads < 1 || n_heads > 1024 || n_seqs < 0 || n_seqs > 65535 || total_q < 0 || total_k < 0 || max_q_len < 0 || max_k_len < 0)
    return fail(IT_INVALID_INPUT, "%s: n_heads %d (1 to 1024), n_seqs %d (to 65535), total_q %d, total_k %d, max_q_len %d, max_k_len %d",
                who, n_heads, n_seqs, total_q, total_k, max_q_len, max_k_len);
  if (nope_dim < 8 || rope_dim < 8 || v_dim < 8 || nope_dim % 8 || rope_dim % 8 || v_dim % 8 || nope_dim + rope_dim > 1024 || v_dim > 1024)
    return fail(IT_INVALID_INPUT, "%s: nope_dim %d, rope_dim %d, v_dim %d: multiples of 8, key and value at most 1024 elements", who,
                nope_dim, rope_dim, v_dim);
  if (!(scale == scale) || std::isinf(scale)) return fail(IT_INVALID_INPUT, "%s: scale is not finite", who);
  if (total_q <= 1) q_stride = 0;  // not used
  if (total_k <= 1) k_stride = v_stride = rope_stride = 0;
  if (n_heads == 1) q_head_stride = k_head_stride = v_head_stride = 0;
  for (int64_t s : {q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride, rope_stride})
    if (s < 0 || s > kFar) return fail(IT_INVALID_INPUT, "%s: stride %lld", who, (long long)s);
  if (n_seqs == 0 || total_q == 0 || max_q_len == 0) return IT_OK;
  if (!q || !out || !cu_q || !cu_k || (total_k && (!k || !v || !k_rope))) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  const int64_t es = dtype_bytes(dtype);
  if (!aligned(q, es) || !aligned(k, es) || !aligned(v, es) || !aligned(k_rope, es) || !aligned(out, 16))
    return fail(IT_INVALID_INPUT, "%s: tensors must be aligned to their elements, out to 16 bytes", who);
  LatentPrefillArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.k_rope = k_rope;
  a.q_stride = q_stride;
  a.q_head = q_head_stride;
  a.k_stride = k_stride;
  a.k_head = k_head_stride;
  a.v_stride = v_stride;
  a.v_head = v_head_stride;
  a.rope_stride = rope_stride;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.out = out;
  a.scale_log2 = scale * kLog2e;
  a.n_heads = n_heads;
  a.nope = nope_dim;
  a.rope = rope_dim;
  a.v_dim = v_dim;
  a.n_seqs = n_seqs;
  a.total_q = total_q;
  a.total_k = total_k;
  a.max_q_len = max_q_len < total_q ? max_q_len : total_q;
  a.max_k_len = max_k_len;
  a.causal = causal != 0;
  a.out_dtype = out_dtype;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (!latent_prefill_matrix(a, dtype, s, e)) {
    const dim3 grid(unsigned(a.max_q_len), unsigned(n_heads), unsigned(n_seqs));
    switch (dtype) {
      case IT_F32: hipLaunchKernelGGL(latent_prefill_general<IT_F32>, grid, dim3(kThreads), 0, s, a); break;
      case IT_BF16: hipLaunchKernelGGL(latent_prefill_general<IT_BF16>, grid, dim3(kThreads), 0, s, a); break;
      default: hipLaunchKernelGGL(latent_prefill_general<IT_F16>, grid, dim3(kThreads), 0, s, a); break;
    }
    e = hipGetLastError();
  }
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
