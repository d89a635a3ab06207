// it_rotary.hip -- rotary positions in either pair layout, over all or part of
// a head, with scaled frequencies: standalone (forwards or transposed) and
// fused into the slot-mapped KV append.
//
//   (a', b') = m (a cos t - b sin t, a sin t + b cos t),  t = pos f_p
//
// The rotation is six operations for each 8 (fp32) or 4 (16-bit) bytes read and
// as many written: bound by memory.  A wave takes one token; its position,
// slot and angles (one pair a lane, shared through LDS) serve all of that
// token's heads, and all its rows are loaded before the first is stored.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>

#include "it_rotary.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxDims = 1024;
constexpr int kQuantV = 4;  // a lane's vector for the quantised formats: 8 lanes of 4 elements own a 32-group

struct RotaryArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  char* kpool;
  char* vpool;
  const int64_t* slots;      // NULL: no cache (rotation only; hkv = 0)
  const int32_t* positions;
  const double* turns;
  uint32_t* err;
  int64_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
  int64_t n_tokens, page_bytes, n_slots;
  float magnitude;
  int hq, hkv, log2_bs, src_dtype, out_dtype, transpose;
  RowSplit split;
};

// Rows of a token: q's heads, then k's, then v's.  SRC: dtype of q, k, v.
// DT: the cache's dtype (SRC where there is no cache).  V: elements of a
// lane's vector (16 bytes of SRC, or four for the quantised formats).
template <int SRC, int DT, int V, int G>
__global__ __launch_bounds__(kThreads) void rotary_rows(RotaryArgs a) {
  using In = RowVec<SRC, V>;
  extern __shared__ __attribute__((aligned(16))) float2 angles[];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = int(threadIdx.x & 63);
  const int64_t t = int64_t(blockIdx.x) * kWaves + wave;
  if (t >= a.n_tokens) return;  // uniform
  const RowSplit& s = a.split;
  const int pairs = s.n_dims >> 1;
  float2* const own = angles + wave * angle_room<V>(s.n_dims);
  const int sub = int((uint32_t(lane) * s.inv) >> 16), c = lane - sub * s.lanes;
  const bool used = sub < s.rows;  // lanes past the wave's last whole row idle
  const int rows = a.hq + 2 * a.hkv;
  const int row0 = int(blockIdx.y) * (s.rows * G) + sub;
  const int pos = a.positions[t];
  const int64_t slot = a.slots ? a.slots[t] : -1;
  // A token at a negative position writes nothing where there is a cache.
  if (a.err && pos < 0) {
    if (blockIdx.y == 0 && lane == 0) atomicOr(a.err, kErrPos);
    return;
  }
  LanePairs<V> lp(s, c);
  typename In::raw xa[G], xb[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    // Past the last row a lane re-reads it; only the stores are predicated.
    const int r = min(row0 + j * s.rows, rows - 1);
    const int rk = r - a.hq, rv = rk - a.hkv;
    const int64_t at = rk < 0 ? t * a.q_stride + int64_t(r) * s.head_dim
                       : rv < 0 ? t * a.k_stride + int64_t(rk) * s.head_dim
                                : t * a.v_stride + int64_t(rv) * s.head_dim;
    const char* const src = static_cast<const char*>(rk < 0 ? a.q : rv < 0 ? a.k : a.v) + at * (SRC == IT_F32 ? 4 : 2);
    const int es = SRC == IT_F32 ? 4 : 2;
    xa[j] = __builtin_nontemporal_load(reinterpret_cast<const typename In::raw*>(src + lp.ea * es));
    xb[j] = __builtin_nontemporal_load(reinterpret_cast<const typename In::raw*>(src + lp.eb * es));
  }
  wave_angles(own, a.turns, pairs, pos, a.magnitude, a.transpose, lane);
  lp.load(s, own);
  if (a.err && slot >= a.n_slots && blockIdx.y == 0 && lane == 0) atomicOr(a.err, kErrSlot);
  const bool cached = slot >= 0 && slot < a.n_slots;  // uniform
  const int64_t blk = slot >> a.log2_bs;
  const int64_t off = slot & ((int64_t(1) << a.log2_bs) - 1);
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int r = row0 + j * s.rows;
    const int rk = r - a.hq, rv = rk - a.hkv;
    if (r >= rows || !used) continue;
    float fa[V], fb[V];
    In::widen(xa[j], fa);
    In::widen(xb[j], fb);
    if (rv < 0) lp.turn(s, fa, fb);
    if (rk < 0) {
      const int64_t at = t * a.out_stride + int64_t(r) * s.head_dim;
      store_row_vec<V>(a.q_out, at + lp.ea, a.out_dtype, fa);
      store_row_vec<V>(a.q_out, at + lp.eb, a.out_dtype, fb);
    } else if (cached) {
      char* const page = (rv < 0 ? a.kpool : a.vpool) + (blk * a.hkv + (rv < 0 ? rk : rv)) * a.page_bytes;
      if constexpr (DT == IT_F32 || DT == IT_BF16 || DT == IT_F16) {
        store_row_vec<V>(page, off * s.head_dim + lp.ea, DT, fa);
        store_row_vec<V>(page, off * s.head_dim + lp.eb, DT, fb);
      } else {
        // The eight lanes of a 32-group hold the same row: all of them are here.
        const int va = lp.ea >> 2, vb = lp.eb >> 2;
        store_group<DT>(page, off, int64_t(1) << a.log2_bs, s.head_dim, va,
                        quant_group<DT>(make_float4(fa[0], fa[1], fa[2], fa[3]), va & 7));
        store_group<DT>(page, off, int64_t(1) << a.log2_bs, s.head_dim, vb,
                        quant_group<DT>(make_float4(fb[0], fb[1], fb[2], fb[3]), vb & 7));
      }
    }
  }
}

// Any even n_dims, head_dim, alignment and stride: one pair, or one element
// past n_dims, per lane (quantised k and v: four elements of a 32-group, whose
// other halves of their pairs are read again).  blockIdx.y: 0 q, 1 k, 2 v.
// Quantised caches come here where a half of the pairs is no multiple of a 32-group:
// 32 of 128 elements or a whole head of 96 in halves.  Bound by its fp64 angles, one
// per element and head: us for 1 / 128 / 4096 tokens of 32 + 2 x 8 bf16 heads of 128,
// 32 of each rotated: Q8_0 4.1 / 7.2 / 174, Q4_0 4.1 / 8.0 / 188, Q5_1 4.3 / 8.8 / 219
// (rotary_rows with all 128: 3.1 / 4.0 / 24.1, 3.0 / 3.6 / 23.3, 3.3 / 3.9 / 25.9; into
// bf16 2.7 / 3.2 / 20.8); 9 + 2 x 3 heads of 96, Q8_0: 3.7 / 4.5 / 35.8.  Rows that are
// not aligned to their vectors, 128 of 128 into bf16: 2.8 / 4.7 / 87.6.
template <int DT>
__global__ __launch_bounds__(kThreads) void rotary_general(RotaryArgs a) {
  const int part = blockIdx.y;
  const int H = part == 0 ? a.hq : a.hkv;
  const int d = a.split.head_dim, nd = a.split.n_dims, half = nd >> 1;
  const bool halves = a.split.layout == IT_ROTARY_HALF;
  constexpr bool kQuant = !(DT == IT_F32 || DT == IT_BF16 || DT == IT_F16);
  const int items = kQuant && part != 0 ? d >> 2 : half + (d - nd);
  const int64_t gid = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const bool live = gid < a.n_tokens * H * items;
  const int64_t th = live ? gid / items : 0;
  const int item = live ? int(gid % items) : int(threadIdx.x % 8);
  const int64_t t = H ? th / H : 0;
  const int h = H ? int(th % H) : 0;
  if (!H) return;  // uniform
  const int pos = a.positions[t];
  const bool pos_ok = !a.err || pos >= 0;
  if (live && !pos_ok && part == 1 && h == 0 && item == 0) atomicOr(a.err, kErrPos);
  const int64_t slot = a.slots ? a.slots[t] : -1;
  if (live && pos_ok && a.err && slot >= a.n_slots && part == 1 && h == 0 && item == 0) atomicOr(a.err, kErrSlot);
  const bool cached = slot >= 0 && slot < a.n_slots;
  const int64_t blk = slot >> a.log2_bs;
  const int64_t off = slot & ((int64_t(1) << a.log2_bs) - 1);
  const void* const src = part == 0 ? a.q : part == 1 ? a.k : a.v;
  const int64_t at = t * (part == 0 ? a.q_stride : part == 1 ? a.k_stride : a.v_stride) + int64_t(h) * d;
  char* const page = (part == 2 ? a.vpool : a.kpool) + (cached ? (blk * a.hkv + h) * a.page_bytes : 0);
  const auto angle = [&](int p) {
    const float2 cs = rotary_angle(a.turns[p], pos);
    return make_float2(cs.x * a.magnitude, (a.transpose ? -cs.y : cs.y) * a.magnitude);
  };
  if constexpr (kQuant) {
    if (part != 0) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (live && pos_ok) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 4 * item + j;
          x[j] = load_element(src, at + e, a.src_dtype);
          if (part == 1 && e < nd) {
            const bool second = halves ? e >= half : (e & 1) != 0;
            const int partner = halves ? (second ? e - half : e + half) : e ^ 1;
            const float2 cs = angle(halves ? (second ? e - half : e) : e >> 1);
            const float y = load_element(src, at + partner, a.src_dtype);
            x[j] = second ? turn_second(cs, y, x[j]) : turn_first(cs, x[j], y);
          }
        }
      }
      // Every lane of a group takes part in its reductions.
      const QuantGroup g = quant_group<DT>(make_float4(x[0], x[1], x[2], x[3]), item & 7);
      if (live && pos_ok && cached) store_group<DT>(page, off, int64_t(1) << a.log2_bs, d, item, g);
      return;
    }
  }
  if (!live || !pos_ok || (part != 0 && !cached)) return;
  void* const out = part == 0 ? a.q_out : page;
  const int64_t to = part == 0 ? t * a.out_stride + int64_t(h) * d : off * d;
  const int dt = part == 0 ? a.out_dtype : DT;
  if (item < half) {
    const int e0 = halves ? item : 2 * item, e1 = halves ? item + half : 2 * item + 1;
    float x = load_element(src, at + e0, a.src_dtype), y = load_element(src, at + e1, a.src_dtype);
    if (part != 2) LanePairs<4>::pair(angle(item), x, y);
    store_element(out, to + e0, dt, x);
    store_element(out, to + e1, dt, y);
  } else {
    const int e = nd + item - half;
    store_element(out, to + e, dt, load_element(src, at + e, a.src_dtype));
  }
}

// Row steps per wave: one, or two where the waves of one would come to four times
// what is resident (32 of 256 CUs).  us with one / two / four, 32 + 2 x 8 heads of
// 128 into a bf16 cache: f32, 1 token 2.41 / 2.81 / 3.58, 1024 8.84 / 9.40 / 9.34, 4096
// (201 MB) 34.8 / 33.1 / 33.7; bf16, 128 tokens 3.01 / 3.50 / 4.43, 1024 5.59 / 5.76 /
// 6.24, 4096 20.7 / 20.8 / 20.8.  Large calls move 5 to 6 TB/s, a copy's rate.
constexpr int64_t kManyWaves = 4 * 256 * 32;

template <int SRC, int DT, int V, int G>
void launch_rows(const RotaryArgs& a, int64_t chunks, hipStream_t s) {
  const dim3 grid(unsigned((a.n_tokens + kWaves - 1) / kWaves), unsigned(chunks));
  hipLaunchKernelGGL((rotary_rows<SRC, DT, V, G>), grid, dim3(kThreads), size_t(kWaves) * angle_room<V>(a.split.n_dims) * sizeof(float2), s, a);
}
template <int SRC, int DT>
void launch_split(const RotaryArgs& a, hipStream_t s) {
  constexpr bool kFloat = DT == IT_F32 || DT == IT_BF16 || DT == IT_F16;
  constexpr int V = kFloat && SRC != IT_F32 ? 8 : 4;
  const int64_t rows = int64_t(a.hq) + 2 * int64_t(a.hkv);
  const auto chunks = [&](int g) { return (rows + a.split.rows * g - 1) / (a.split.rows * g); };
  if (a.n_tokens * chunks(1) <= kManyWaves) launch_rows<SRC, DT, V, 1>(a, chunks(1), s);
  else launch_rows<SRC, DT, V, 2>(a, chunks(2), s);
}
template <int DT>
void launch_general(const RotaryArgs& a, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL(rotary_general<DT>, dim3(unsigned(blocks), a.hkv ? 3 : 1), dim3(kThreads), 0, s, a);
}
template <int SRC>
void launch_src(const RotaryArgs& a, int cache_dtype, hipStream_t s) {
  switch (cache_dtype) {
    case IT_F32: return launch_split<SRC, IT_F32>(a, s);
    case IT_BF16: return launch_split<SRC, IT_BF16>(a, s);
    case IT_F16: return launch_split<SRC, IT_F16>(a, s);
    case IT_Q4_0: return launch_split<SRC, IT_Q4_0>(a, s);
    case IT_Q4_1: return launch_split<SRC, IT_Q4_1>(a, s);
    case IT_Q5_0: return launch_split<SRC, IT_Q5_0>(a, s);
    case IT_Q5_1: return launch_split<SRC, IT_Q5_1>(a, s);
    default: return launch_split<SRC, IT_Q8_0>(a, s);
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool is_float(int32_t dt) { return dt == IT_F32 || dt == IT_F16 || dt == IT_BF16; }

// Rows of n tokens: byte range [lo, hi).
struct Span {
  uintptr_t lo, hi;
  Span(const void* p, int64_t n, int64_t stride, int64_t row, int64_t es)
      : lo(reinterpret_cast<uintptr_t>(p)), hi(lo + uintptr_t(((n - 1) * stride + row) * es)) {}
  bool overlaps(const Span& o) const { return lo < o.hi && o.lo < hi; }
};

// Picks the kernel and launches on `device`.  a.split holds head_dim, n_dims
// and layout; cache_dtype the destination's (the source's where none).
int32_t launch(RotaryArgs& a, int32_t cache_dtype, int32_t device, void* stream, const char* who) {
  const int64_t es = dtype_bytes(a.src_dtype), oes = dtype_bytes(a.out_dtype);
  const bool quant = is_quant(cache_dtype);
  const int v = quant || a.src_dtype == IT_F32 ? kQuantV : 8;
  const int d = a.split.head_dim, nd = a.split.n_dims;
  // Vectors of v elements at addresses aligned to them, 16 bytes at most.
  const auto vec_ok = [&](const void* p, int64_t stride, int64_t e) {
    return !p || (aligned(p, uintptr_t(v * e < 16 ? v * e : 16)) && stride % v == 0);
  };
  const bool fast = row_split(d, nd, a.split.layout, v, quant ? 32 : v, a.split) && vec_ok(a.q, a.q_stride, es) &&
                    vec_ok(a.k, a.k_stride, es) && vec_ok(a.v, a.v_stride, es) && vec_ok(a.q_out, a.out_stride, oes);
  const int64_t rows = int64_t(a.hq) + 2 * int64_t(a.hkv);
  int64_t blocks;
  if (fast) {
    blocks = (a.n_tokens + kWaves - 1) / kWaves;
    if ((rows + a.split.rows - 1) / a.split.rows > 65535) return fail(IT_INVALID_INPUT, "%s: too many heads", who);
  } else {
    const int64_t h = a.hq > a.hkv ? a.hq : a.hkv, items = quant ? d : nd / 2 + (d - nd);
    if (a.n_tokens > (int64_t(1) << 40) / (h * items)) return fail(IT_INVALID_INPUT, "%s: too many tokens", who);
    blocks = (a.n_tokens * h * items + kThreads - 1) / kThreads;
  }
  // A grid has fewer than 2^32 work items in each direction.
  if (blocks >= (int64_t(1) << 32) / kThreads) return fail(IT_INVALID_INPUT, "%s: too many tokens", who);
  int dev = -1;
  (void)hipGetDevice(&dev);
  if (dev != device) (void)hipSetDevice(device);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!fast) {
    switch (cache_dtype) {
      case IT_F32: launch_general<IT_F32>(a, blocks, s); break;
      case IT_BF16: launch_general<IT_BF16>(a, blocks, s); break;
      case IT_F16: launch_general<IT_F16>(a, blocks, s); break;
      case IT_Q4_0: launch_general<IT_Q4_0>(a, blocks, s); break;
      case IT_Q4_1: launch_general<IT_Q4_1>(a, blocks, s); break;
      case IT_Q5_0: launch_general<IT_Q5_0>(a, blocks, s); break;
      case IT_Q5_1: launch_general<IT_Q5_1>(a, blocks, s); break;
      default: launch_general<IT_Q8_0>(a, blocks, s); break;
    }
  } else if (a.src_dtype == IT_F32) {
    launch_src<IT_F32>(a, cache_dtype, s);
  } else if (a.src_dtype == IT_BF16) {
    launch_src<IT_BF16>(a, cache_dtype, s);
  } else {
    launch_src<IT_F16>(a, cache_dtype, s);
  }
  const hipError_t e = hipGetLastError();
  if (dev >= 0 && dev != device) (void)hipSetDevice(dev);
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
}  // namespace

// ---------------------------------------------------------------------------
// The handle.
// ---------------------------------------------------------------------------
extern "C" int32_t it_rotary_frequencies(const it_rotary_desc* d, double* freqs) {
  const char* who = "it_rotary_frequencies";
  if (!d || !freqs) return fail(IT_INVALID_INPUT, "%s: NULL argument", who);
  if (d->n_dims <= 0 || d->n_dims % 2 || d->n_dims > kMaxDims)
    return fail(IT_INVALID_INPUT, "%s: n_dims %d must be even, in [2, %d]", who, d->n_dims, kMaxDims);
  const int pairs = d->n_dims / 2;
  if (d->inv_freq) {
    for (int p = 0; p < pairs; ++p) freqs[p] = d->inv_freq[p];
  } else {
    if (!(d->freq_base > 0.0) || !std::isfinite(d->freq_base))
      return fail(IT_INVALID_INPUT, "%s: freq_base must be positive and finite", who);
    if (d->scaling < IT_ROTARY_SCALE_NONE || d->scaling > IT_ROTARY_SCALE_PARTS)
      return fail(IT_NOT_IMPLEMENTED, "%s: scaling %d", who, d->scaling);
    const double s = d->scaling == IT_ROTARY_SCALE_NONE ? 1.0 : d->factor;
    if (!(s > 0.0) || !std::isfinite(s)) return fail(IT_INVALID_INPUT, "%s: factor must be positive and finite", who);
    const bool parts = d->scaling == IT_ROTARY_SCALE_PARTS;
    if (parts && (d->original_ctx <= 0 || !(d->low >= 0.0) || !(d->high > d->low) || !std::isfinite(d->high)))
      return fail(IT_INVALID_INPUT, "%s: scaling by parts needs original_ctx > 0 and 0 <= low < high", who);
    double base = d->freq_base;
    // The base that stretches the slowest pair's wavelength `factor` times and leaves the fastest as it is.
    if (d->scaling == IT_ROTARY_SCALE_BASE && d->n_dims > 2) base *= std::pow(s, double(d->n_dims) / (d->n_dims - 2));
    for (int p = 0; p < pairs; ++p) {
      double f = std::pow(base, -2.0 * p / d->n_dims);
      if (d->scaling == IT_ROTARY_SCALE_LINEAR) f /= s;
      if (parts) {
        const double turns = d->original_ctx * f / 6.283185307179586;
        double g = (turns - d->low) / (d->high - d->low);
        g = g < 0.0 ? 0.0 : g > 1.0 ? 1.0 : g;
        f *= g + (1.0 - g) / s;
      }
      freqs[p] = f;
    }
  }
  for (int p = 0; p < pairs; ++p)
    if (!std::isfinite(freqs[p]) || std::fabs(freqs[p]) > 1048576.0)
      return fail(IT_INVALID_INPUT, "%s: frequency %d must be finite, at most 2^20", who, p);
  return IT_OK;
}

extern "C" int32_t it_rotary_new(int32_t device, const it_rotary_desc* d, it_rotary** out) {
  const char* who = "it_rotary_new";
  if (!out) return fail(IT_INVALID_INPUT, "%s: out is NULL", who);
  *out = nullptr;
  double freqs[kMaxDims / 2], turns[kMaxDims / 2];
  if (int32_t rc = it_rotary_frequencies(d, freqs)) return rc;
  if (d->layout != IT_ROTARY_INTERLEAVED && d->layout != IT_ROTARY_HALF)
    return fail(IT_NOT_IMPLEMENTED, "%s: layout %d", who, d->layout);
  if (!(d->magnitude > 0.0) || !std::isfinite(float(d->magnitude)))
    return fail(IT_INVALID_INPUT, "%s: magnitude must be positive and finite", who);
  const int pairs = d->n_dims / 2;
  const size_t bytes = size_t(pairs) * sizeof(double);
  for (int p = 0; p < pairs; ++p) turns[p] = freqs[p] / 6.283185307179586;
  int prev = -1;
  (void)hipGetDevice(&prev);
  if (hipSetDevice(device) != hipSuccess) {
    (void)hipGetLastError();
    return fail(IT_DEVICE_ERROR, "%s: hipSetDevice(%d)", who, device);
  }
  double* dev = nullptr;
  hipError_t e = hipMalloc(&dev, bytes);
  if (e == hipSuccess) e = hipMemcpy(dev, turns, bytes, hipMemcpyHostToDevice);
  auto* r = new (std::nothrow) it_rotary{dev, float(d->magnitude), device, d->n_dims, d->layout};
  if (e != hipSuccess || !r) {
    if (dev) (void)hipFree(dev);
    if (prev >= 0) (void)hipSetDevice(prev);
    delete r;
    return fail(IT_DEVICE_ERROR, "%s: %s", who, e != hipSuccess ? hipGetErrorString(e) : "out of host memory");
  }
  if (prev >= 0) (void)hipSetDevice(prev);
  *out = r;
  return IT_OK;
}

extern "C" int32_t it_rotary_destroy(it_rotary* r) {
  if (!r) return IT_OK;
  int prev = -1;
  (void)hipGetDevice(&prev);
  (void)hipSetDevice(r->device);
  const hipError_t e = hipFree(r->turns);
  if (prev >= 0) (void)hipSetDevice(prev);
  delete r;
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "it_rotary_destroy: %s", hipGetErrorString(e));
}

// ---------------------------------------------------------------------------
// Rotation alone.
// ---------------------------------------------------------------------------
extern "C" int32_t it_rotary_apply(const it_rotary* rotary, const void* x, int32_t dtype, int64_t token_stride,
                                   const int32_t* positions, int32_t n_tokens, int32_t n_heads, int32_t head_dim,
                                   int32_t transpose, void* out, int64_t out_stride, void* stream) {
  const char* who = "it_rotary_apply";
  if (!rotary) return fail(IT_INVALID_INPUT, "%s: rotary is NULL", who);
  if (!is_float(dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: dtype %d (F32, F16 or BF16)", who, dtype);
  if (n_tokens < 0 || n_heads <= 0 || head_dim <= 0 || head_dim > 65536 || n_heads > 65536)
    return fail(IT_INVALID_INPUT, "%s: shape [%d][%d][%d]", who, n_tokens, n_heads, head_dim);
  if (rotary->n_dims > head_dim)
    return fail(IT_INVALID_INPUT, "%s: %d rotated elements > head_dim %d", who, rotary->n_dims, head_dim);
  const int64_t row = int64_t(n_heads) * head_dim, es = dtype_bytes(dtype), kFar = int64_t(1) << 40;
  if (n_tokens > 1 && (token_stride < row || out_stride < row || token_stride > kFar || out_stride > kFar))
    return fail(IT_INVALID_INPUT, "%s: strides %lld, %lld below a token's %lld elements (or above 2^40)", who,
                (long long)token_stride, (long long)out_stride, (long long)row);
  if (n_tokens == 0) return IT_OK;
  if (n_tokens == 1) token_stride = out_stride = row;  // not used
  if (!x || !out || !positions) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  if (!aligned(x, uintptr_t(es)) || !aligned(out, uintptr_t(es)))
    return fail(IT_INVALID_INPUT, "%s: tensors must be aligned to their elements", who);
  const bool same = x == out && token_stride == out_stride;
  if (!same && Span(x, n_tokens, token_stride, row, es).overlaps(Span(out, n_tokens, out_stride, row, es)))
    return fail(IT_INVALID_INPUT, "%s: out overlaps x (out may be x itself, with its stride)", who);
  RotaryArgs a{};
  a.q = x;
  a.q_out = out;
  a.positions = positions;
  a.turns = rotary->turns;
  a.q_stride = token_stride;
  a.out_stride = out_stride;
  a.n_tokens = n_tokens;
  a.magnitude = rotary->magnitude;
  a.hq = n_heads;
  a.src_dtype = a.out_dtype = dtype;
  a.transpose = transpose != 0;
  a.split.head_dim = head_dim;
  a.split.n_dims = rotary->n_dims;
  a.split.layout = rotary->layout;
  return launch(a, dtype, rotary->device, stream, who);
}

// ---------------------------------------------------------------------------
// Rotation and append.
// ---------------------------------------------------------------------------
extern "C" int32_t it_kv_append_rotary(it_kv_cache* c, const it_rotary* rotary, const void* q, const void* k, const void* v,
                                       int32_t src_dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                       int32_t n_heads, const int64_t* slot_mapping, const int32_t* positions,
                                       int32_t n_tokens, void* q_out, int32_t q_out_dtype, void* stream) {
  const char* who = "it_kv_append_rotary";
  if (!c || !rotary) return fail(IT_INVALID_INPUT, "%s: cache or rotary is NULL", who);
  if (int32_t rc = one_layer(c, who)) return rc;
  if (int32_t rc = per_head(c, who)) return rc;
  if (!is_float(src_dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: src_dtype %d (F32, F16 or BF16)", who, src_dtype);
  if (n_tokens < 0) return fail(IT_INVALID_INPUT, "%s: n_tokens %d < 0", who, n_tokens);
  if (n_heads < 0 || n_heads > 65536 || n_heads % c->n_kv_heads)
    return fail(IT_INVALID_INPUT, "%s: n_heads %d must be a multiple of n_kv_heads %d (0: no q)", who, n_heads, c->n_kv_heads);
  if (c->n_kv_heads > 65536) return fail(IT_NOT_IMPLEMENTED, "%s: %d KV heads", who, c->n_kv_heads);
  if (n_heads && !is_float(q_out_dtype)) return fail(IT_NOT_IMPLEMENTED, "%s: q_out dtype %d (F32, F16 or BF16)", who, q_out_dtype);
  if (rotary->n_dims > c->head_dim)
    return fail(IT_INVALID_INPUT, "%s: %d rotated elements > head_dim %d", who, rotary->n_dims, c->head_dim);
  if (rotary->device != c->device) return fail(IT_INVALID_INPUT, "%s: rotary and cache on different devices", who);
  const int64_t qrow = int64_t(n_heads) * c->head_dim, kvrow = int64_t(c->n_kv_heads) * c->head_dim;
  const int64_t es = dtype_bytes(src_dtype), kFar = int64_t(1) << 40;
  if (n_tokens > 1 && (q_stride < qrow || k_stride < kvrow || v_stride < kvrow || q_stride > kFar || k_stride > kFar || v_stride > kFar))
    return fail(IT_INVALID_INPUT, "%s: strides %lld, %lld, %lld below a token's %lld, %lld elements (or above 2^40)", who,
                (long long)q_stride, (long long)k_stride, (long long)v_stride, (long long)qrow, (long long)kvrow);
  if (n_tokens == 0) return IT_OK;
  if (n_tokens == 1) q_stride = qrow, k_stride = v_stride = kvrow;  // not used
  if (!k || !v || !slot_mapping || !positions || (n_heads && (!q || !q_out))) return fail(IT_INVALID_INPUT, "%s: NULL tensor", who);
  const int64_t oes = n_heads ? dtype_bytes(q_out_dtype) : 4;
  if (!aligned(k, uintptr_t(es)) || !aligned(v, uintptr_t(es)) ||
      (n_heads && (!aligned(q, uintptr_t(es)) || !aligned(q_out, uintptr_t(oes)))))
    return fail(IT_INVALID_INPUT, "%s: tensors must be aligned to their elements", who);
  if (n_heads) {
    const Span o(q_out, n_tokens, qrow, qrow, oes);
    const bool same = q_out == q && q_out_dtype == src_dtype && q_stride == qrow;
    if ((!same && o.overlaps(Span(q, n_tokens, q_stride, qrow, es))) || o.overlaps(Span(k, n_tokens, k_stride, kvrow, es)) ||
        o.overlaps(Span(v, n_tokens, v_stride, kvrow, es)))
      return fail(IT_INVALID_INPUT, "%s: q_out overlaps q, k or v (it may be q itself, contiguous and of its dtype)", who);
  }
  RotaryArgs a{};
  a.q = n_heads ? q : nullptr;
  a.k = k;
  a.v = v;
  a.q_out = n_heads ? q_out : nullptr;
  a.kpool = static_cast<char*>(c->k_pool);
  a.vpool = static_cast<char*>(c->v_pool);
  a.slots = slot_mapping;
  a.positions = positions;
  a.turns = rotary->turns;
  a.err = c->err_flag;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.out_stride = qrow;
  a.n_tokens = n_tokens;
  a.page_bytes = c->page_bytes;
  a.n_slots = c->num_blocks * c->block_size;
  a.magnitude = rotary->magnitude;
  a.hq = n_heads;
  a.hkv = c->n_kv_heads;
  a.log2_bs = c->log2_bs;
  a.src_dtype = src_dtype;
  a.out_dtype = n_heads ? q_out_dtype : IT_F32;
  a.split.head_dim = c->head_dim;
  a.split.n_dims = rotary->n_dims;
  a.split.layout = rotary->layout;
  return launch(a, c->dtype, c->device, stream, who);
}
