// it_move.hip -- token rows moved between slots of a paged cache, in every
// layer and head, keys turned to their new positions on the way: what drops
// tokens out of the middle of a sequence and gives their pages back.
//
// K is cached rotated by its position p; at position p + delta it must be
// R(p + delta) k = R(delta) R(p) k, so one more rotation of the cached row is
// all that is needed.  Bound by memory: each row of K and V is read and written
// once.  A wave takes one (src, dst) pair and a run of its rows (layers x heads
// x {K, V}), all loaded before the first is stored; its angles are computed
// once.  A source row is one run of head_dim elements, consecutive pairs'
// destination rows are neighbours in a page, so both sides move whole sectors.
#include <hip/hip_runtime.h>

#include "it_rotary.hpp"

using namespace itkv;

namespace {
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

struct MoveArgs {
  char* kpool;
  char* vpool;
  const int64_t* src;
  const int64_t* dst;
  const int32_t* delta;  // NULL: copy
  const double* turns;
  uint32_t* err;
  int64_t n, n_slots, page_bytes, layer_bytes;
  uint32_t heads, rows;  // rows of a pair: layers x heads x pools moved
  int log2_bs;
  int main_bytes, side_bytes;  // of a token's row in a page; the side row is quantised formats' (scales, high bits)
  int pools;                   // 2: K then V; 1: V alone (byte copies), K alone (quantised keys), latent rows
  int latent;                  // elements of a latent row before its rope part
  RowSplit split;
};

// A pair's slots; false: nothing to do.  Slots out of range are latched.
__device__ __forceinline__ bool move_slots(const MoveArgs& a, int64_t i, int64_t& s, int64_t& d, bool latch) {
  s = a.src[i];
  d = a.dst[i];
  if (s < 0 || d < 0) return false;
  if (s >= a.n_slots || d >= a.n_slots) {
    if (latch) atomicOr(a.err, kErrSlot);
    return false;
  }
  return true;
}
// The page that holds row r of a slot: layer-major, then K's heads, then V's.
__device__ __forceinline__ char* move_page(const MoveArgs& a, uint32_t r, int64_t slot, bool& key) {
  const uint32_t per = a.heads * uint32_t(a.pools);
  const uint32_t layer = r / per, x = r - layer * per;
  key = a.pools == 2 && x < a.heads;
  const uint32_t h = x < a.heads ? x : x - a.heads;
  return (key ? a.kpool : a.vpool) + layer * a.layer_bytes + ((slot >> a.log2_bs) * a.heads + h) * a.page_bytes;
}

// Rows as they are: 16-byte pieces of the main row, then 2-byte ones of the
// side row, which take quantised copies away from a copy's rate (4096 rows of 28
// layers x 4 heads of 128: bf16 70.9 us, 6.6 TB/s; Q8_0 55.6, 4.5; Q4_0 40.3, 3.3; Q4_1
// 51.0, 2.9; Q5_0 64.8, 2.5; Q5_1 73.7, 2.4).
__global__ __launch_bounds__(kThreads) void kv_move_bytes(MoveArgs a) {
  const int64_t i = int64_t(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
  if (i >= a.n) return;  // uniform
  const int lane = int(threadIdx.x & 63);
  int64_t s, d;
  if (!move_slots(a, i, s, d, blockIdx.y == 0 && lane == 0) || s == d) return;  // uniform
  const uint32_t vecs = uint32_t(a.main_bytes) >> 4, items = vecs + (uint32_t(a.side_bytes) >> 1), total = a.rows * items;
  const int64_t bs = int64_t(1) << a.log2_bs, so = s & (bs - 1), dof = d & (bs - 1);
  const uint32_t x = blockIdx.y * 64 + uint32_t(lane);
  if (x >= total) return;
  const uint32_t r = x / items, item = x - r * items;
  bool key;
  const char* const from = move_page(a, r, s, key);
  char* const to = move_page(a, r, d, key);
  if (item < vecs) {
    st16(to + dof * a.main_bytes + item * 16, ld16_nt(from + so * a.main_bytes + item * 16));
  } else {
    const int64_t side = bs * a.main_bytes + (item - vecs) * 2;
    *reinterpret_cast<uint16_t*>(to + side + dof * a.side_bytes) = *reinterpret_cast<const uint16_t*>(from + side + so * a.side_bytes);
  }
}

// F32, F16 and BF16 rows, K turned.
template <int DT, int G>
__global__ __launch_bounds__(kThreads) void kv_move_rows(MoveArgs a) {
  constexpr int V = DT == IT_F32 ? 4 : 8;
  constexpr int kBytes = DT == IT_F32 ? 4 : 2;
  using Row = RowVec<DT, V>;
  extern __shared__ __attribute__((aligned(16))) float2 angles[];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = int(threadIdx.x & 63);
  const int64_t i = int64_t(blockIdx.x) * kWaves + wave;
  if (i >= a.n) return;  // uniform
  int64_t s, d;
  if (!move_slots(a, i, s, d, blockIdx.y == 0 && lane == 0)) return;  // uniform
  const int delta = a.delta[i];
  if (s == d && delta == 0) return;
  const RowSplit& sp = a.split;
  const int pairs = sp.n_dims >> 1;
  float2* const own = angles + wave * angle_room<V>(sp.n_dims);
  const int sub = int((uint32_t(lane) * sp.inv) >> 16), c = lane - sub * sp.lanes;
  const bool used = sub < sp.rows;
  const int64_t bs = int64_t(1) << a.log2_bs, so = s & (bs - 1), dof = d & (bs - 1);
  const uint32_t row0 = blockIdx.y * uint32_t(sp.rows * G) + uint32_t(sub);
  LanePairs<V> lp(sp, c);
  typename Row::raw xa[G], xb[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const uint32_t r = min(row0 + uint32_t(j * sp.rows), a.rows - 1);  // past the end: re-read, not stored
    bool key;
    const char* const row = move_page(a, r, s, key) + so * a.main_bytes;
    xa[j] = __builtin_nontemporal_load(reinterpret_cast<const typename Row::raw*>(row + lp.ea * kBytes));
    xb[j] = __builtin_nontemporal_load(reinterpret_cast<const typename Row::raw*>(row + lp.eb * kBytes));
  }
  wave_angles(own, a.turns, pairs, delta, 1.0f, false, lane);
  lp.load(sp, own);
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const uint32_t r = row0 + uint32_t(j * sp.rows);
    if (r >= a.rows || !used) continue;
    bool key;
    char* const row = move_page(a, r, d, key) + dof * a.main_bytes;
    // A row that keeps its position keeps its bytes, NaNs and infinities too.
    if (key && delta != 0) {
      float fa[V], fb[V];
      Row::widen(xa[j], fa);
      Row::widen(xb[j], fb);
      lp.turn(sp, fa, fb);
      xa[j] = Row::narrow(fa);
      xb[j] = Row::narrow(fb);
    }
    __builtin_nontemporal_store(xa[j], reinterpret_cast<typename Row::raw*>(row + lp.ea * kBytes));
    __builtin_nontemporal_store(xb[j], reinterpret_cast<typename Row::raw*>(row + lp.eb * kBytes));
  }
}

// The same for rows that cannot be split into vectors with their pairs: a
// pair, or an element past n_dims, per lane.
template <int DT>
__global__ __launch_bounds__(kThreads) void kv_move_general(MoveArgs a) {
  const int nd = a.split.n_dims, half = nd >> 1, items = half + (a.split.head_dim - nd);
  const int64_t gid = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (gid >= a.n * int64_t(a.rows) * items) return;
  const int item = int(gid % items);
  const int64_t ir = gid / items, i = ir / a.rows;
  const uint32_t r = uint32_t(ir - i * a.rows);
  int64_t s, d;
  if (!move_slots(a, i, s, d, r == 0 && item == 0)) return;
  const int delta = a.delta[i];
  const int64_t bs = int64_t(1) << a.log2_bs;
  bool key;
  const char* const from = move_page(a, r, s, key) + (s & (bs - 1)) * a.main_bytes;
  char* const to = move_page(a, r, d, key) + (d & (bs - 1)) * a.main_bytes;
  if (s == d && (!key || delta == 0)) return;
  typedef std::conditional_t<DT == IT_F32, uint32_t, uint16_t> bits;
  const auto copy = [&](int e) { reinterpret_cast<bits*>(to)[e] = reinterpret_cast<const bits*>(from)[e]; };
  if (item >= half) return copy(nd + item - half);
  const bool halves = a.split.layout == IT_ROTARY_HALF;
  const int e0 = halves ? item : 2 * item, e1 = halves ? item + half : 2 * item + 1;
  if (!key || delta == 0) {
    copy(e0);
    copy(e1);
    return;
  }
  float x = load_element(from, e0, DT), y = load_element(from, e1, DT);
  LanePairs<4>::pair(rotary_angle(a.turns[item], delta), x, y);
  store_element(to, e0, DT, x);
  store_element(to, e1, DT, y);
}

// Latent rows, their rope part turned: a wave takes one (pair, layer) row, the
// latent as 16-byte pieces, a lane per pair of the rope part.  Each lane writes
// what it has read itself, so a row may be turned in place.
template <int DT>
__global__ __launch_bounds__(kThreads) void kv_move_latent(MoveArgs a) {
  const int lane = int(threadIdx.x & 63);
  const int64_t i = int64_t(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (i >= a.n) return;
  int64_t s, d;
  if (!move_slots(a, i, s, d, blockIdx.y == 0 && lane == 0)) return;
  const int delta = a.delta[i], half = a.split.n_dims >> 1;
  const int64_t bs = int64_t(1) << a.log2_bs;
  if (s == d && delta == 0) return;
  bool key;
  const char* const from = move_page(a, blockIdx.y, s, key) + (s & (bs - 1)) * a.main_bytes;
  char* const to = move_page(a, blockIdx.y, d, key) + (d & (bs - 1)) * a.main_bytes;
  const bool halves = a.split.layout == IT_ROTARY_HALF;
  const int pieces = a.latent * (DT == IT_F32 ? 4 : 2) / 16;
  for (int p = lane; p < half; p += 64) {
    const int e0 = a.latent + (halves ? p : 2 * p), e1 = a.latent + (halves ? p + half : 2 * p + 1);
    float x = load_element(from, e0, DT), y = load_element(from, e1, DT);
    if (delta) LanePairs<4>::pair(rotary_angle(a.turns[p], delta), x, y);
    store_element(to, e0, DT, x);
    store_element(to, e1, DT, y);
  }
  if (s == d) return;
  for (int p = lane; p < pieces; p += 64) st16(to + p * 16, ld16(from + p * 16));
}

// Elements 4 cv .. 4 cv + 3 of a quantised token row.
template <int DT>
__device__ __forceinline__ float4 dequant4(const char* page, int64_t off, int64_t bs, int d, int cv) {
  const int g = cv >> 3, l8 = cv & 7;
  float x[4];
  if constexpr (DT == IT_Q8_0) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(page + off * d + cv * 4);
    const float sc = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(page + bs * d + (off * (d >> 5) + g) * 2));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = sc * float(int32_t(w << (24 - 8 * j)) >> 24);
  } else {
    using N = NibFmt<DT>;
    const int ng = d >> 5;
    const char* const side = page + bs * (d >> 1) + off * (ng * N::kSide);
    // Byte j of the group holds elements j (low nibble) and j + 16 (high).
    const uint32_t w = *reinterpret_cast<const uint32_t*>(page + off * (d >> 1) + g * 16 + (l8 & 3) * 4) >> (l8 < 4 ? 0 : 4);
    uint32_t high = 0u;
    if constexpr (N::kQ5) high = *reinterpret_cast<const uint32_t*>(side + 4 * g) >> (4 * l8);
    float sc, base;
    if constexpr (N::kMin) {
      const uint32_t m = *reinterpret_cast<const uint32_t*>(side + N::meta_off(ng) + 4 * g);
      sc = f16_bits_to_f32(m & 0xFFFFu);
      base = f16_bits_to_f32(m >> 16);
    } else {
      sc = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(side + N::meta_off(ng) + 2 * g));
      base = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int q = int((w >> (8 * j)) & 0xFu);
      if constexpr (N::kQ5) q |= int((high >> j) & 1u) << 4;
      if constexpr (!N::kMin) q -= N::kQ5 ? 16 : 8;
      x[j] = N::kMin ? mul_rn(sc, float(q)) + base : sc * float(q);
    }
  }
  return make_float4(x[0], x[1], x[2], x[3]);
}

// Quantised K rows, turned: a wave dequantises a row into LDS, turns it there
// pair by pair's elements and quantises it again.  The whole row is read before
// any of it is written (src may be dst).  Bound by latency: a row's loads, its two
// LDS stages and its stores follow one another, with half the lanes idle at head_dim
// 128.  us for 16 / 2000 / 4096 rows of 28 layers x 4 heads of 128, with V's copy: Q8_0
// 6.6 / 103 / 194 (1.3 TB/s), Q4_0 6.5 / 101 / 190, Q4_1 6.6 / 113 / 216, Q5_0 6.7 / 116
// / 222, Q5_1 6.8 / 129 / 246 (0.7); bf16 (kv_move_rows) 3.8 / 41 / 84 (5.6).
template <int DT>
__global__ __launch_bounds__(kThreads) void kv_move_quant(MoveArgs a) {
  extern __shared__ __attribute__((aligned(16))) float2 angles[];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = int(threadIdx.x & 63);
  const int64_t i = int64_t(blockIdx.x) * kWaves + wave;
  if (i >= a.n) return;  // uniform
  int64_t s, d;
  if (!move_slots(a, i, s, d, blockIdx.y == 0 && lane == 0)) return;  // uniform
  const int delta = a.delta[i];
  if (s == d && delta == 0) return;
  const int dim = a.split.head_dim, nd = a.split.n_dims, half = nd >> 1, vecs = dim >> 2;
  const bool halves = a.split.layout == IT_ROTARY_HALF;
  float2* const cs = angles + wave * (half + (dim >> 1));
  float* const row = reinterpret_cast<float*>(cs + half);
  wave_angles(cs, a.turns, half, delta, 1.0f, false, lane);
  const int64_t bs = int64_t(1) << a.log2_bs, so = s & (bs - 1), dof = d & (bs - 1);
  for (uint32_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    bool key;
    const char* const from = move_page(a, r, s, key);
    char* const to = move_page(a, r, d, key);
    if (delta == 0) {  // keeps its bytes
      const int main = a.main_bytes >> 2, side = a.side_bytes >> 1;
      for (int x = lane; x < main; x += 64)
        reinterpret_cast<uint32_t*>(to + dof * a.main_bytes)[x] = reinterpret_cast<const uint32_t*>(from + so * a.main_bytes)[x];
      for (int x = lane; x < side; x += 64)
        reinterpret_cast<uint16_t*>(to + bs * a.main_bytes + dof * a.side_bytes)[x] =
            reinterpret_cast<const uint16_t*>(from + bs * a.main_bytes + so * a.side_bytes)[x];
      continue;
    }
    for (int cv = lane; cv < vecs; cv += 64) {
      const float4 x = dequant4<DT>(from, so, bs, dim, cv);
      row[4 * cv] = x.x;
      row[4 * cv + 1] = x.y;
      row[4 * cv + 2] = x.z;
      row[4 * cv + 3] = x.w;
    }
    wave_lds_fence();
    for (int cv = lane; cv < vecs; cv += 64) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * cv + j;
        x[j] = row[e];
        if (e < nd) {
          const bool second = halves ? e >= half : (e & 1) != 0;
          const float y = row[halves ? (second ? e - half : e + half) : e ^ 1];
          const float2 t = cs[halves ? (second ? e - half : e) : e >> 1];
          x[j] = second ? turn_second(t, y, x[j]) : turn_first(t, x[j], y);
        }
      }
      // dim % 32 == 0: the eight lanes of a 32-group are all here.
      store_group<DT>(to, dof, bs, dim, cv, quant_group<DT>(make_float4(x[0], x[1], x[2], x[3]), cv & 7));
    }
    wave_lds_fence();
  }
}

void launch_bytes(const MoveArgs& a, hipStream_t s) {
  // One 16-byte piece per lane: two or four were slower at every size but one (28
  // layers x 4 heads of 128 bf16: 16 tokens 2.20 us, 2.55 with two, 2000 35.2, 36.0).
  const int64_t total = int64_t(a.rows) * (a.main_bytes / 16 + a.side_bytes / 2);
  hipLaunchKernelGGL(kv_move_bytes, dim3(unsigned((a.n + kWaves - 1) / kWaves), unsigned((total + 63) / 64)), dim3(kThreads), 0, s, a);
}

// Row steps per wave: one, or two where the waves of one would come to four times
// what is resident (32 of 256 CUs), which shares a token's angles among more rows.
// us with one / two / four, 28 layers x 4 heads of 128 bf16: 16 tokens 2.92 / 3.40 /
// 4.11, 260 6.4 / 6.4 / 5.9, 2000 39.2 / 38.1 / 39.5 (6 TB/s from a warm cache).
constexpr int64_t kManyWaves = 4 * 256 * 32;

template <int DT>
void launch_rows(const MoveArgs& a, bool split, hipStream_t s) {
  if (!split) {
    const int64_t items = a.split.n_dims / 2 + (a.split.head_dim - a.split.n_dims);
    const int64_t blocks = (a.n * int64_t(a.rows) * items + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(kv_move_general<DT>, dim3(unsigned(blocks)), dim3(kThreads), 0, s, a);
    return;
  }
  const size_t lds = size_t(kWaves) * angle_room<DT == IT_F32 ? 4 : 8>(a.split.n_dims) * sizeof(float2);
  const auto chunks = [&](int g) { return (int64_t(a.rows) + a.split.rows * g - 1) / (a.split.rows * g); };
  const unsigned bx = unsigned((a.n + kWaves - 1) / kWaves);
  if (a.n * chunks(1) <= kManyWaves)
    hipLaunchKernelGGL((kv_move_rows<DT, 1>), dim3(bx, unsigned(chunks(1))), dim3(kThreads), lds, s, a);
  else
    hipLaunchKernelGGL((kv_move_rows<DT, 2>), dim3(bx, unsigned(chunks(2))), dim3(kThreads), lds, s, a);
}
void launch_latent(const MoveArgs& a, int32_t dtype, hipStream_t s) {
  auto* const kern = dtype == IT_F32 ? kv_move_latent<IT_F32> : dtype == IT_BF16 ? kv_move_latent<IT_BF16> : kv_move_latent<IT_F16>;
  hipLaunchKernelGGL(kern, dim3(unsigned((a.n + kWaves - 1) / kWaves), a.rows), dim3(kThreads), 0, s, a);
}
template <int DT>
void launch_quant(MoveArgs a, hipStream_t s) {
  // K alone: its heads are the only ones of a layer (the pool that move_page
  // takes for one pool is vpool).
  a.rows /= 2;
  a.pools = 1;
  char* const v = a.vpool;
  a.vpool = a.kpool;
  const size_t lds = size_t(kWaves) * (a.split.n_dims / 2 + a.split.head_dim / 2) * sizeof(float2);
  // A wave per row, rows beyond what is resident one after another.
  const int64_t want = 256 * 32 / a.n, y = want < 1 ? 1 : want > int64_t(a.rows) ? int64_t(a.rows) : want;
  hipLaunchKernelGGL(kv_move_quant<DT>, dim3(unsigned((a.n + kWaves - 1) / kWaves), unsigned(y < 65535 ? y : 65535)),
                     dim3(kThreads), lds, s, a);
  a.vpool = v;
  launch_bytes(a, s);
}
}  // namespace

extern "C" int32_t it_kv_move(it_kv_cache* c, const int64_t* src, const int64_t* dst, int32_t n, const it_rotary* rotary,
                              const int32_t* delta, void* stream) {
  const char* who = "it_kv_move";
  if (!c) return fail(IT_INVALID_INPUT, "%s: cache is NULL", who);
  if (n < 0) return fail(IT_INVALID_INPUT, "%s: n %d < 0", who, n);
  if (rotary && c->latent_dim && rotary->n_dims != c->head_dim - c->latent_dim)
    return fail(IT_INVALID_INPUT, "%s: %d rotated elements, a latent row turns its %d rope elements", who, rotary->n_dims,
                c->head_dim - c->latent_dim);
  if (rotary && rotary->n_dims > c->head_dim)
    return fail(IT_INVALID_INPUT, "%s: %d rotated elements > head_dim %d", who, rotary->n_dims, c->head_dim);
  if (rotary && rotary->device != c->device) return fail(IT_INVALID_INPUT, "%s: rotary and cache on different devices", who);
  const bool quant = is_quant(c->dtype);
  if (rotary && quant && c->head_dim > 1024) return fail(IT_NOT_IMPLEMENTED, "%s: quantised rows of %d elements", who, c->head_dim);
  if (n == 0) return IT_OK;
  if (!src || !dst) return fail(IT_INVALID_INPUT, "%s: NULL slots", who);
  if (rotary && !delta) return fail(IT_INVALID_INPUT, "%s: delta is NULL", who);
  const int pools = c->latent_dim ? 1 : 2;
  const int64_t rows = int64_t(c->n_layers) * c->n_kv_heads * pools, row_items = int64_t(c->head_dim) * 2;
  // A pair's rows are chunks of a grid's second direction (fewer than 65536 at
  // this limit: a chunk is 64 pieces of 16 bytes or 2), pairs its first (2^32 work
  // items).
  if (rows * row_items >= int64_t(1) << 24 || n > 1 << 25)
    return fail(IT_INVALID_INPUT, "%s: %d pairs of %lld rows of %d elements", who, n, (long long)rows, c->head_dim);
  MoveArgs a{};
  a.kpool = static_cast<char*>(c->k_pool);
  a.vpool = static_cast<char*>(c->latent_dim ? c->k_pool : c->v_pool);
  a.latent = c->latent_dim;
  a.src = src;
  a.dst = dst;
  a.delta = rotary ? delta : nullptr;
  a.turns = rotary ? rotary->turns : nullptr;
  a.err = c->err_flag;
  a.n = n;
  a.n_slots = c->num_blocks * c->block_size;
  a.page_bytes = c->page_bytes;
  a.layer_bytes = c->layer_bytes;
  a.heads = uint32_t(c->n_kv_heads);
  a.rows = uint32_t(rows);
  a.log2_bs = c->log2_bs;
  const int64_t row_bytes = c->page_bytes / c->block_size;
  a.main_bytes = int(c->dtype == IT_Q8_0 ? c->head_dim : quant ? c->head_dim / 2 : row_bytes);
  a.side_bytes = int(row_bytes - a.main_bytes);
  a.pools = pools;
  bool split = false;
  if (rotary && !c->latent_dim) {
    a.split.head_dim = c->head_dim;
    a.split.n_dims = rotary->n_dims;
    a.split.layout = rotary->layout;
    const int v = c->dtype == IT_F32 ? 4 : 8;
    if (!quant) split = row_split(c->head_dim, rotary->n_dims, rotary->layout, v, v, a.split);
    if (!quant && !split && int64_t(n) * rows >= (int64_t(1) << 32) / c->head_dim)
      return fail(IT_INVALID_INPUT, "%s: %d pairs of %lld rows of %d elements", who, n, (long long)rows, c->head_dim);
  }
  int dev = -1;
  (void)hipGetDevice(&dev);
  if (dev != c->device) (void)hipSetDevice(c->device);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!rotary) {
    launch_bytes(a, s);
  } else if (c->latent_dim) {
    a.split.head_dim = c->head_dim;
    a.split.n_dims = rotary->n_dims;
    a.split.layout = rotary->layout;
    launch_latent(a, c->dtype, s);
  } else {
    switch (c->dtype) {
      case IT_F32: launch_rows<IT_F32>(a, split, s); break;
      case IT_BF16: launch_rows<IT_BF16>(a, split, s); break;
      case IT_F16: launch_rows<IT_F16>(a, split, s); break;
      case IT_Q4_0: launch_quant<IT_Q4_0>(a, s); break;
      case IT_Q4_1: launch_quant<IT_Q4_1>(a, s); break;
      case IT_Q5_0: launch_quant<IT_Q5_0>(a, s); break;
      case IT_Q5_1: launch_quant<IT_Q5_1>(a, s); break;
      default: launch_quant<IT_Q8_0>(a, s); break;
    }
  }
  const hipError_t e = hipGetLastError();
  if (dev >= 0 && dev != c->device) (void)hipSetDevice(dev);
  return e == hipSuccess ? IT_OK : fail(IT_DEVICE_ERROR, "%s: launch: %s", who, hipGetErrorString(e));
}
