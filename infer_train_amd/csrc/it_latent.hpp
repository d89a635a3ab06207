// it_latent.hpp -- latent attention: what its kernels share.
#pragma once
#include <hip/hip_runtime.h>

#include "it_internal.hpp"
#include "it_kv.h"

namespace itkv {

// Absorbed attention of q_len new tokens of each sequence over its cached rows.
struct LatentDecodeArgs {
  const void* q_latent;
  const void* q_rope;
  int64_t ql_stride, ql_head, qr_stride, qr_head;  // elements between tokens and heads
  const char* pool;
  const int32_t* bt;
  const int32_t* ctx_lens;
  const int32_t* start_pos;  // NULL: 0
  void* out;
  uint32_t* err;
  float* ws;
  int64_t page_bytes, num_blocks;
  float scale_log2;  // scale * log2(e)
  int n_heads, q_len, n_seqs, max_blocks, max_tokens, log2_bs;
  int latent, rope;
  int out_dtype;
};

// Expanded attention.
struct LatentPrefillArgs {
  const void *q, *k, *v, *k_rope;
  int64_t q_stride, q_head, k_stride, k_head, v_stride, v_head, rope_stride;
  const int32_t *cu_q, *cu_k;
  void* out;
  float scale_log2;
  int n_heads, nope, rope, v_dim, n_seqs, total_q, total_k, max_q_len, max_k_len, causal, out_dtype;
};

// Whether a sequence's rows and keys lie in the tensors and under the bounds.
__device__ __forceinline__ bool latent_prefill_fits(const LatentPrefillArgs& a, int q0, int q1, int k0, int k1) {
  return q0 >= 0 && q1 >= q0 && q1 <= a.total_q && q1 - q0 <= a.max_q_len && k0 >= 0 && k1 >= k0 && k1 <= a.total_k &&
         k1 - k0 <= a.max_k_len;
}

// A sequence's keys as a decode sees them: [start, ctx), empty where a length or
// start is not one (latched where a block may write `err`).
struct LatentSpan {
  int start, ctx;
};
__device__ __forceinline__ LatentSpan latent_span(const LatentDecodeArgs& a, int b, bool latch) {
  const int ctx = a.ctx_lens[b], st = a.start_pos ? a.start_pos[b] : 0;
  if (ctx <= 0 || st >= ctx) return {0, 0};
  uint32_t bad = 0u;
  if (st < 0) bad = kErrStart;
  else if (ctx - (st & ~31) > a.max_tokens) bad = kErrCtx;
  else if ((ctx - 1) >> a.log2_bs >= a.max_blocks) bad = kErrTable;
  if (bad) {
    if (latch) atomicOr(a.err, bad);
    return {0, 0};
  }
  return {st, ctx};
}

constexpr int kLatentNarrow = 288;  // elements of a row of which LDS holds two tiles for each of four token groups
constexpr int kLatentMaxQ = 64;  // new tokens of a sequence

// How an absorbed call's tokens are divided, and where pieces of sequences go.
struct LatentSplitPlan {
  int workers;   // runs that the tiles are divided into
  int row_wgs;   // workgroups that share a run, each with QG * 16 queries of its own
  float4* o;     // partial O^T: [worker][row wg][2][QG][L / 16][64 lanes]
  float2* ml;    // and its (maximum, sum): [worker][row wg][2][QG][16]
  int2* shares;  // of each sequence that holds something: its first worker and how many share it
};

hipError_t latent_decode_bf16(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s);
hipError_t latent_decode_f16(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s);

// The matrix-core kernels: false where they do not take the call (its type,
// widths or pages); else launched, `e` the result.  n_cu: the device's compute
// units (latent_compute_units).
int latent_compute_units(int device);
size_t latent_decode_matrix_ws(int32_t dtype, int latent, int rope, int block_size, int n_seqs, int q_len, int n_heads, int max_tokens,
                               int n_cu);
bool latent_decode_matrix(const LatentDecodeArgs& a, int32_t dtype, int block_size, int n_cu, hipStream_t s, hipError_t& e);
bool latent_prefill_matrix(const LatentPrefillArgs& a, int32_t dtype, hipStream_t s, hipError_t& e);

}  // namespace itkv
