/*
 * it_kv.h -- C ABI of the MI355X (gfx950) KV-cache hot path.
 *
 * This is the drop-in boundary for InferTrain's KV-cache path.  Every entry
 * point is `extern "C"`, takes plain pointers, sizes and a HIP stream passed
 * as `void*`, and returns a status code that mirrors the reference's OpError
 * (src/types.rs:227-231).  No call aborts: conditions the reference asserts
 * on (src/backend/arm/flash_attn.rs:16-19, quant.rs:150) return
 * IT_INVALID_INPUT, and it_last_error() holds a thread-local message.
 *
 * Memory: every tensor argument of a device entry point (it_kv_*, it_paged_*,
 * it_flash_attention) is DEVICE memory owned by the caller; work is enqueued
 * on `stream` and returns without synchronising.  Host-side objects
 * (it_block_pool, it_kv_manager) take host memory.  Device-side checks that
 * cannot be made before launch (a slot or block id out of range in a device
 * array) never fault: the access is skipped or clamped, and the condition is
 * latched in the cache and reported by it_kv_cache_check().
 *
 * dtype codes are the ggml QuantType ids of src/types.rs:106-144.
 */
#ifndef IT_KV_H
#define IT_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes: OpError (src/types.rs:227-231) ----------------------- */
#define IT_OK 0
#define IT_NOT_IMPLEMENTED 1 /* OpError::NotImplemented */
#define IT_INVALID_INPUT 2   /* OpError::InvalidInput  */
#define IT_DEVICE_ERROR 3    /* OpError::DeviceError   */

/* ---- dtype codes: QuantType (src/types.rs:106-144) ---------------------- */
#define IT_F32 0
#define IT_F16 1
#define IT_Q4_0 2
#define IT_Q4_1 3
#define IT_Q5_0 6
#define IT_Q5_1 7
#define IT_Q8_0 8
#define IT_BF16 30

#define IT_BLOCK_SIZE 16        /* src/memory/paged.rs:9, default page size */
#define IT_QK8_0 32             /* src/types.rs:11 */
#define IT_BLOCK_Q8_0_BYTES 34  /* sizeof(BlockQ8_0), src/types.rs:34-41,250 */
#define IT_QK4_0 32             /* src/types.rs:7 */
#define IT_BLOCK_Q4_0_BYTES 18  /* sizeof(BlockQ4_0), src/types.rs:15-22 */
#define IT_QK4_1 32             /* src/types.rs:8 */
#define IT_BLOCK_Q4_1_BYTES 20  /* sizeof(BlockQ4_1), src/types.rs:24-32,249 */
#define IT_QK5_0 32             /* src/types.rs:9 */
#define IT_BLOCK_Q5_0_BYTES 22  /* ggml block_q5_0 {u16 d; u8 qh[4]; u8 qs[16]}: the reference has the
                                   type id (types.rs:116) and no struct */
#define IT_QK5_1 32             /* src/types.rs:10 */
#define IT_BLOCK_Q5_1_BYTES 24  /* ggml block_q5_1 {u16 d; u16 m; u8 qh[4]; u8 qs[16]} (types.rs:117) */

/* ---- operator ids for it_supports (Backend::supports_op/_quant,
 *      src/backend.rs:184-186) ------------------------------------------- */
#define IT_OP_KV_APPEND 1
#define IT_OP_KV_GATHER 2
#define IT_OP_KV_EVICT 3
#define IT_OP_PAGED_DECODE 4
#define IT_OP_PAGED_PREFILL 5
#define IT_OP_FLASH_ATTENTION 6 /* CoreOperator::FlashAttention, src/types.rs:202-208 */
#define IT_OP_KV_COPY_BLOCKS 7
#define IT_OP_KV_APPEND_ROTARY 8 /* dtype: the cache's */
#define IT_OP_ROTARY 9           /* dtype: the tensor's */
#define IT_OP_KV_MOVE 10         /* dtype: the cache's */
#define IT_OP_SAMPLE 11          /* dtype: the logits' */
#define IT_OP_LATENT_APPEND 12   /* dtype: the latent cache's */
#define IT_OP_LATENT_DECODE 13   /* dtype: the latent cache's */
#define IT_OP_LATENT_PREFILL 14  /* dtype: q's, k's and v's */
#define IT_OP_BEAM_SELECT 15     /* dtype: the logits' */
#define IT_OP_BEAM_REORDER 16    /* any dtype: whole bytes are moved */

/* Thread-local message for the last non-OK status on this thread. */
const char* it_last_error(void);
int32_t it_abi_version(void);
/* 1 if (op, dtype) is implemented, else 0.  dtype is the cache dtype. */
int32_t it_supports(int32_t op, int32_t dtype);

/* ======================================================================== */
/* Host: block allocator.  Replaces memory::paged::BlockPool                */
/* (src/memory/paged.rs:21-58).                                              */
/* ======================================================================== */
typedef struct it_block_pool it_block_pool;

/* BlockPool::new (paged.rs:28-34): free list 0..capacity, refcounts 0. */
int32_t it_block_pool_new(int64_t capacity, int32_t quant_type, it_block_pool** out);
/* As new, but the free list is `order` (a permutation of 0..capacity-1),
 * bottom to top, so the first allocate returns order[capacity-1]. */
int32_t it_block_pool_new_ordered(const int64_t* order, int64_t capacity, int32_t quant_type,
                                  it_block_pool** out);
void it_block_pool_destroy(it_block_pool* pool);
/* BlockPool::allocate (paged.rs:36-42): LIFO pop, refcount 1; -1 = None. */
int64_t it_block_pool_allocate(it_block_pool* pool);
/* BlockPool::share (paged.rs:44-46), with one departure: the reference
 * increments the refcount of any block, a free one included, which leaves
 * that block on the free list and referenced at once (the next allocate
 * would hand out a live block).  Here sharing a free block (refcount 0) is
 * IT_INVALID_INPUT and changes nothing. */
int32_t it_block_pool_share(it_block_pool* pool, int64_t id);
/* BlockPool::free (paged.rs:48-53); a free at refcount 0 (a u32 underflow
 * in the reference) is IT_INVALID_INPUT. */
int32_t it_block_pool_free(it_block_pool* pool, int64_t id);
/* BlockPool::quant_type (paged.rs:55-57). */
int32_t it_block_pool_quant_type(const it_block_pool* pool);
int64_t it_block_pool_num_free(const it_block_pool* pool);
int64_t it_block_pool_capacity(const it_block_pool* pool);
/* Refcount of `id`, -1 if out of range. */
int64_t it_block_pool_ref_count(const it_block_pool* pool, int64_t id);

/* ======================================================================== */
/* Host: slot mapping, block tables and sliding-window eviction.  The        */
/* reference batcher (src/batcher/continuous.rs:28-74) only admits requests; */
/* this is the per-step state it lacks.                                      */
/*   slot(pos) = table[pos / block_size] * block_size + pos % block_size     */
/*   a block is allocated from the pool when pos % block_size == 0           */
/*   window W > 0: before the token at position p, every held block whose    */
/*   last position is < p - W + 1 is released with BlockPool::free, oldest   */
/*   first; sequences are processed in the order the caller lists them.      */
/* Block tables are indexed by absolute logical block (pos / block_size).    */
/* ======================================================================== */
typedef struct it_kv_manager it_kv_manager;

/* The manager borrows `pool`; the pool must outlive it. window 0 = none. */
int32_t it_kv_manager_new(it_block_pool* pool, int32_t block_size, int32_t max_seqs,
                          int32_t max_blocks_per_seq, int32_t window, it_kv_manager** out);
void it_kv_manager_destroy(it_kv_manager* mgr);
/* Make sequence `seq` hold `blocks` (already allocated from the pool) as
 * logical blocks first_block.., with the next token at position `pos`. */
int32_t it_kv_manager_seed_seq(it_kv_manager* mgr, int32_t seq, int64_t pos, int64_t first_block,
                               const int32_t* blocks, int32_t n_blocks);
/* One step's plan, filled by it_kv_manager_step.  The caller owns every
 * array; a NULL pointer marks an output it does not want.
 * Blocks "released" by a sequence drop that sequence's reference
 * (BlockPool::free, paged.rs:48-53); only those whose refcount reaches 0
 * return to the pool.  `evicted` lists exactly those, in free order: the
 * pages to clear with it_kv_evict.  A block that another (forked) sequence
 * still holds is released but not listed, and its pages stay intact.
 * Returned blocks go back on the pool's free list when the step ends, in
 * free order, so within one step no block is both freed and handed out
 * again.  A token whose block the window returns later in the same step
 * (a step that appends more tokens than the window holds) gets slot -1:
 * it is never written.
 * Device order of a step: it_kv_copy_blocks(cow_src, cow_dst), then
 * it_kv_evict(evicted), then the append, then it_kv_sync_tables; a copy
 * source the same step returns to the pool is read before it is cleared. */
typedef struct {
  int64_t* slots;      /* [tokens_cap] slot of every new token, in list order */
  int32_t* token_seq;  /* [tokens_cap] its sequence, or NULL (it_kv_sync_tables' seq) */
  int32_t* token_pos;  /* [tokens_cap] its position, or NULL (it_kv_sync_tables' pos) */
  int32_t tokens_cap;
  int32_t n_tokens;    /* out: sum(n_tokens) */
  int32_t* evicted;    /* [evicted_cap] blocks returned to the pool by the window */
  int32_t evicted_cap;
  int32_t n_evicted;   /* out */
  int32_t* cow_src;    /* [cow_cap] copy-on-write pairs (page copies to make  */
  int32_t* cow_dst;    /*   before the append); cow_src NULL = no copy-on-write */
  int32_t cow_cap;
  int32_t n_cow;       /* out */
  int32_t* ctx_lens;   /* [max_seqs] after the step (next position), or NULL */
  int32_t* start_pos;  /* [max_seqs] after the step (window start, else 0), or NULL */
} it_kv_step_plan;

/* Append n_tokens[i] tokens to seqs[i], in list order (a sequence may be
 * listed more than once), and fill `plan`.  Sequence ids, counts and
 * tokens_cap are checked before any state changes; a later error (pool
 * exhausted, a capacity exceeded) leaves the manager state unspecified.
 * No counterpart in the reference: its batcher (continuous.rs:28-74)
 * admits requests but builds no slot mapping; this is that step. */
int32_t it_kv_manager_step(it_kv_manager* mgr, const int32_t* seqs, const int32_t* n_tokens,
                           int32_t n, it_kv_step_plan* plan);
/* it_kv_manager_step with slots (sized sum(n_tokens)) and the evicted list
 * only. */
int32_t it_kv_manager_append(it_kv_manager* mgr, const int32_t* seqs, const int32_t* n_tokens,
                             int32_t n, int64_t* slots_out, int32_t* evicted_out,
                             int32_t evicted_cap, int32_t* n_evicted);
/* Release every block of `seq` (BlockPool::free, lowest logical block
 * first) and reset it to position 0.  The blocks that return to the pool
 * (refcount 0) go to evicted_out; evicted_cap must cover every block the
 * sequence holds, else IT_INVALID_INPUT and nothing changes. */
int32_t it_kv_manager_release_seq(it_kv_manager* mgr, int32_t seq, int32_t* evicted_out,
                                  int32_t evicted_cap, int32_t* n_evicted);
/* Prefix sharing: dst takes src's blocks and position; each block gets
 * BlockPool::share (paged.rs:44-46).  dst must be empty.  The first append
 * to a shared partial block copies it (copy-on-write): the manager
 * allocates a fresh block and reports the (src, dst) pair in cow_out. */
int32_t it_kv_manager_fork(it_kv_manager* mgr, int32_t src_seq, int32_t dst_seq);
/* it_kv_manager_step with copy-on-write, slots, evicted and cow lists. */
int32_t it_kv_manager_append_cow(it_kv_manager* mgr, const int32_t* seqs, const int32_t* n_tokens,
                                 int32_t n, int64_t* slots_out, int32_t* evicted_out,
                                 int32_t evicted_cap, int32_t* n_evicted, int32_t* cow_src,
                                 int32_t* cow_dst, int32_t cow_cap, int32_t* n_cow);
/* Compact sequence `seq` to the tokens at the positions keep[0..n_keep)
 * (ascending, each below the sequence's next position): keep[i] becomes
 * position i and n_keep the next position.  Leading blocks whose tokens all
 * keep their positions stay as they are (dropping only a tail, as after a
 * rejected draft, moves nothing); from the first other block on, kept rows go
 * to fresh blocks, so that forks of the sequence are untouched and no row is
 * overwritten before it is read.  A last block that stays may be a fork's too,
 * with tokens beyond n_keep that the fork still reads: the next append to the
 * sequence then has to copy it (it_kv_manager_append_cow, or a step with
 * cow_src), and one without copy-on-write is IT_INVALID_INPUT before any state
 * changes (it_kv_manager_needs_cow).  The caller then runs, in this order:
 * it_kv_move(src, dst, delta), it_kv_evict(evicted), it_kv_sync_tables(seq,
 * pos, dst), all of it queued before the device work of any later call of the
 * manager: the returned blocks are the next that the pool hands out, to an
 * append or to another compaction.  So plans of two calls are not joined into
 * one move; it_kv_manager_compact_many plans several sequences for one.
 *   src, dst: int64[moves_cap] slots of the moved rows; delta: new - old
 *     position of each (NULL = not wanted); pos: new position (NULL likewise);
 *     *n_moves of them (at most n_keep)
 *   evicted: blocks that returned to the pool (refcount 0), *n_evicted of them
 * IT_INVALID_INPUT, and nothing changes, where a capacity does not suffice,
 * the pool holds too few free blocks, or a kept position is not held; for a
 * manager with a window IT_NOT_IMPLEMENTED: its blocks go by position. */
int32_t it_kv_manager_compact(it_kv_manager* mgr, int32_t seq, const int32_t* keep, int32_t n_keep,
                              int64_t* src, int64_t* dst, int32_t* delta, int32_t* pos, int32_t moves_cap,
                              int32_t* n_moves, int32_t* evicted, int32_t evicted_cap, int32_t* n_evicted);
/* it_kv_manager_compact of several sequences as one plan: of seqs[i], keep
 * [cu_keep[i] .. cu_keep[i + 1]) stays (cu_keep: n_seqs + 1 values from 0; each
 * sequence once).  No destination is a source, or a returned block, of any of
 * them, so that one it_kv_move, one it_kv_evict and one it_kv_sync_tables
 * (token_seq, pos, dst) serve all.  moves_cap, evicted_cap and the free blocks
 * that are needed are sums over the sequences; token_seq, delta and pos may be
 * NULL.  IT_INVALID_INPUT and nothing changes, for any of them, as above. */
int32_t it_kv_manager_compact_many(it_kv_manager* mgr, const int32_t* seqs, int32_t n_seqs, const int32_t* keep,
                                   const int32_t* cu_keep, int64_t* src, int64_t* dst, int32_t* delta,
                                   int32_t* token_seq, int32_t* pos, int32_t moves_cap, int32_t* n_moves,
                                   int32_t* evicted, int32_t evicted_cap, int32_t* n_evicted);
/* 1: one append of tokens to each of seqs[0..n) needs copy-on-write, because a
 * compaction set the position of one back to where another sequence holds a
 * token in the same block, or where another of seqs would write one, or a
 * reordering left several to continue a block; 0: it does not; -1: an argument
 * is invalid. */
int32_t it_kv_manager_needs_cow(const it_kv_manager* mgr, const int32_t* seqs, int32_t n);
/* Beams reordered: sequence seqs[i] becomes what seqs[parents[i]] was before
 * the call (parents[i] an index into the list; below 0, or i itself: it stays),
 * so that one parent may be continued by several and another by none.  Blocks
 * are shared, none is copied: the next append to these sequences has to be
 * copy-on-write, as after it_kv_manager_fork, and a device block table's rows
 * are put in the same order (it_beam_reorder).  seqs: distinct.
 *   evicted: blocks that returned to the pool (no sequence continues them), in
 *     the order of the list and of their positions: the pages to clear with
 *     it_kv_evict; evicted_cap must cover every block that the sequences hold
 *     (each once), else IT_INVALID_INPUT
 * IT_INVALID_INPUT changes nothing. */
int32_t it_kv_manager_reorder(it_kv_manager* mgr, const int32_t* seqs, const int32_t* parents, int32_t n,
                              int32_t* evicted, int32_t evicted_cap, int32_t* n_evicted);
/* Export tables [max_seqs][max_blocks] (-1 = not held), ctx_lens[max_seqs]
 * (= next position) and start_pos[max_seqs] (window start, else 0).  Any
 * output pointer may be NULL. */
int32_t it_kv_manager_tables(const it_kv_manager* mgr, int32_t* tables, int32_t max_blocks,
                             int32_t* ctx_lens, int32_t* start_pos);

/* ======================================================================== */
/* Device: the paged cache.  Replaces ForwardExecutor's contiguous           */
/* kv_cache_k/kv_cache_v (src/inference/forward.rs:16-19, 31-37).            */
/* Layout per pool (one for K, one for V), HBM:                              */
/*   [num_blocks][n_kv_heads] pages; a page holds block_size token rows.     */
/*   F32/F16/BF16 page: [block_size][head_dim] elements.                     */
/*   Q8_0 page: int8 qs[block_size][head_dim], then fp16 d[block_size]       */
/*   [head_dim/32] (structure of arrays of BlockQ8_0, src/types.rs:34-41).   */
/*   Q4_0 page: u8 qs[block_size][head_dim/2] (each 32-group's 16 bytes as   */
/*   in BlockQ4_0: low nibble = element j, high = element j+16), then fp16   */
/*   d[block_size][head_dim/32] (src/types.rs:15-22).                        */
/*   Q4_1 page: the Q4_0 nibble plane, then fp16 (d, m) pairs                */
/*   [block_size][head_dim/32] (BlockQ4_1, src/types.rs:24-32).              */
/*   Q5_0 / Q5_1 page: the Q4_0 nibble plane (the low four bits of each      */
/*   5-bit value), then per token a side row: head_dim/32 u32 qh words (bit  */
/*   e = bit 4 of element e, as ggml's block_q5_*), then head_dim/32 fp16 d  */
/*   (Q5_0) or (d, m) pairs (Q5_1).                                          */
/* ======================================================================== */
typedef struct it_kv_cache it_kv_cache;

typedef struct {
  void* k_pool;        /* device */
  void* v_pool;        /* device */
  int64_t num_blocks;
  int64_t page_bytes;  /* bytes of one (block, head) page */
  int32_t block_size;  /* power of two */
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t dtype;
  int32_t device;
  int32_t owns_memory;
  int32_t n_layers;    /* layers in each pool (1 for a layer view) */
} it_kv_cache_desc;

int64_t it_kv_page_bytes(int32_t block_size, int32_t head_dim, int32_t dtype);
/* Allocates both pools on `device` (hipMalloc) and zero-fills them. */
int32_t it_kv_cache_new(int32_t device, int64_t num_blocks, int32_t block_size,
                        int32_t n_kv_heads, int32_t head_dim, int32_t dtype, it_kv_cache** out);
/* Wraps caller-owned pools (num_blocks * n_kv_heads * page_bytes each,
 * 16-byte aligned).  The cache never frees them. */
int32_t it_kv_cache_wrap(int32_t device, void* k_pool, void* v_pool, int64_t num_blocks,
                         int32_t block_size, int32_t n_kv_heads, int32_t head_dim, int32_t dtype,
                         it_kv_cache** out);
/* Every layer of a model in one cache: the reference's per-layer
 * kv_cache_k/kv_cache_v (forward.rs:17-18, 36-37, indexed by layer_idx at
 * :224-228).  Each pool holds n_layers (1..4096) layers one after another,
 * [n_layers][num_blocks][n_kv_heads] pages, so one block id (one manager,
 * one block table) names the same pages in every layer.  it_kv_evict and
 * it_kv_copy_blocks on a multi-layer cache act on every layer in one
 * launch; it_kv_sync_tables and it_kv_cache_check take it as it is.  The
 * per-layer entry points (append, append_rope, gather, decode, prefill)
 * take a layer's view from it_kv_cache_layer and return IT_INVALID_INPUT
 * for a multi-layer handle. */
int32_t it_kv_cache_new_layers(int32_t device, int32_t n_layers, int64_t num_blocks, int32_t block_size,
                               int32_t n_kv_heads, int32_t head_dim, int32_t dtype, it_kv_cache** out);
/* Wraps caller-owned pools of n_layers * num_blocks * n_kv_heads * page_bytes
 * bytes each. */
int32_t it_kv_cache_wrap_layers(int32_t device, int32_t n_layers, void* k_pool, void* v_pool,
                                int64_t num_blocks, int32_t block_size, int32_t n_kv_heads,
                                int32_t head_dim, int32_t dtype, it_kv_cache** out);
/* A one-layer view of layer `layer` (no allocation on the device: the
 * view's pools point into the parent's, and it shares the parent's
 * latched-error word).  Destroy views before their parent. */
int32_t it_kv_cache_layer(const it_kv_cache* cache, int32_t layer, it_kv_cache** out);
int32_t it_kv_cache_destroy(it_kv_cache* cache);
int32_t it_kv_cache_describe(const it_kv_cache* cache, it_kv_cache_desc* out);
/* Synchronises `stream`, then reports (and clears) a latched device-side
 * error: a slot, block id or block-table entry out of range seen by an
 * earlier kernel on this cache.  IT_OK if none. */
int32_t it_kv_cache_check(it_kv_cache* cache, void* stream);

/* KV append: k_cache[slot/bs][h][slot%bs][:] = k[t][h][:], likewise v
 * (forward.rs:219-229 with seq_pos generalised to a slot mapping).
 *   k, v: [n_tokens][n_kv_heads][head_dim] of src_dtype, device.
 *   slot_mapping: int64[n_tokens], device; slot < 0 = padding, skipped.
 * F32/F16/BF16 caches take src_dtype == cache dtype (bit copy).  A Q8_0
 * cache takes F32 and quantises each 32-group exactly as
 * quantize_row_q8_0 (src/backend/arm/quant.rs:149-183).  A Q4_0 cache takes
 * F32 and quantises as ggml's quantize_row_q4_0_ref (the reference has the
 * block and its dequantisation, vec_dot.rs:425-440, but no quantiser).  A
 * Q4_1 cache takes F32 and quantises as ggml's quantize_row_q4_1_ref (the
 * reference has only the block).  Q5_0 / Q5_1 caches take F32 and quantise
 * as ggml's quantize_row_q5_0_ref / quantize_row_q5_1_ref (the reference has
 * only the type ids, types.rs:116-117). */
int32_t it_kv_append(it_kv_cache* cache, const void* k, const void* v, int32_t src_dtype,
                     const int64_t* slot_mapping, int32_t n_tokens, void* stream);

/* RoPE then append (forward.rs:195-229): rope_f32 (src/backend/arm/rope.rs:
 * 6-44) of every q and k head row at its token's position, then the rotated
 * k and the unrotated v into the cache as it_kv_append stores them.
 * The rotation's cos/sin come from `rope`, a table built once on the host
 * with the C library's float32 powf/cosf/sinf in rope_f32's order
 * (theta = (float)pos * powf(freq_base, -(float)i / n_dims) for each even
 * i < n_dims), so device results equal rope_f32's bit for bit.  Elements
 * past n_dims are not rotated (forward.rs passes n_dims = head_dim).
 *   q: F32 [n_tokens][n_heads][head_dim]; k, v: F32 [n_tokens][n_kv_heads][head_dim]
 *   positions: int32[n_tokens] in [0, max_pos) (else latched; the token writes nothing)
 *   slot_mapping: as it_kv_append (slot < 0 = padding: q still rotated)
 *   q_out: [n_tokens][n_heads][head_dim] of q_out_dtype: F32, or the cache
 *          dtype for BF16/F16 caches (round to nearest even)
 * F32 caches store the rotated fp32 values; BF16/F16 caches round them to
 * nearest even; Q8_0 / Q4_0 / Q4_1 / Q5_0 / Q5_1 caches quantise them as
 * it_kv_append does. */
typedef struct it_rope_table it_rope_table;
/* n_dims: a multiple of 4 up to 4096; positions [0, max_pos); device memory
 * max_pos * n_dims * 4 bytes. */
int32_t it_rope_table_new(int32_t device, int32_t n_dims, float freq_base, int32_t max_pos,
                          it_rope_table** out);
int32_t it_rope_table_destroy(it_rope_table* rope);
int32_t it_kv_append_rope(it_kv_cache* cache, const it_rope_table* rope, const float* q, int32_t n_heads,
                          const float* k, const float* v, const int64_t* slot_mapping,
                          const int32_t* positions, int32_t n_tokens, void* q_out, int32_t q_out_dtype,
                          void* stream);

/* ---- rotary positions ---------------------------------------------------
 * The rotation models train with, in either pair layout, over all or part of
 * a head, with frequencies scaled for contexts longer than those trained on:
 *   (a', b') = magnitude * (a cos t - b sin t, a sin t + b cos t),
 *   t = position * f_p   (pair p < n_dims / 2, f_p = freq_base^(-2 p / n_dims))
 * it_kv_append_rope beside it reproduces rope_f32 (src/backend/arm/rope.rs:
 * 6-44) bit for bit from a table; this one holds no table, takes any int32
 * position, and rounds once: the angle is taken in 64 bits, its cosine and sine
 * are each within about one fp32 unit in the last place.  No counterpart in
 * the reference beyond rope_f32's interleaved, unscaled pairs. */
#define IT_ROTARY_INTERLEAVED 0 /* pair p: elements 2p, 2p + 1 (rope_f32) */
#define IT_ROTARY_HALF 1        /* pair p: elements p, p + n_dims / 2 */
#define IT_ROTARY_SCALE_NONE 0
#define IT_ROTARY_SCALE_LINEAR 1 /* position interpolation: f / factor */
#define IT_ROTARY_SCALE_BASE 2   /* freq_base * factor^(n_dims / (n_dims - 2)) */
#define IT_ROTARY_SCALE_PARTS 3  /* by parts: with r = original_ctx * f / (2 pi) turns over the trained
                                    context and g = (r - low) / (high - low) clamped to [0, 1],
                                    f * (g + (1 - g) / factor): the blend is linear in the turns,
                                    as the YaRN paper has it; checkpoints whose code blends linearly
                                    in the pair's index p give their own inv_freq */
typedef struct {
  int32_t n_dims;        /* rotated elements of a head, the first ones: even, 2 .. 1024 */
  int32_t layout;        /* IT_ROTARY_INTERLEAVED, IT_ROTARY_HALF */
  int32_t scaling;       /* IT_ROTARY_SCALE_* */
  int32_t original_ctx;  /* PARTS: positions trained on */
  double freq_base;
  double factor;         /* LINEAR, BASE, PARTS: > 0 */
  double low, high;      /* PARTS: turns below which f / factor, above which f */
  double magnitude;      /* > 0; 1 for a plain rotation (YaRN: 0.1 ln factor + 1) */
  const double* inv_freq; /* NULL, or host double[n_dims / 2]: the f_p themselves, radians per
                             position (freq_base, scaling and what goes with it unused) */
} it_rotary_desc;
typedef struct it_rotary it_rotary;
/* f_p of every pair (host arithmetic, no device): freqs[n_dims / 2]. */
int32_t it_rotary_frequencies(const it_rotary_desc* desc, double* freqs);
/* Device memory: 8 bytes per pair. */
int32_t it_rotary_new(int32_t device, const it_rotary_desc* desc, it_rotary** out);
int32_t it_rotary_destroy(it_rotary* rotary);
/* out = R(position) x for every head of every token; transpose != 0: the
 * transposed rotation, magnitude * R(-position) -- the gradient of the forward
 * one, and with magnitude 1 its inverse.
 *   x, out: [n_tokens][n_heads][head_dim] of dtype F32, F16 or BF16, with
 *     token_stride / out_stride elements between tokens (at least a token's
 *     own; not read for one token); out may be x itself with its stride, and
 *     must not overlap it otherwise
 *   positions: int32[n_tokens], device; any value, negative ones too
 * Products in fp32, rounded once to dtype; elements past n_dims pass through.
 * 16-byte aligned rows run fastest; others are taken too. */
int32_t it_rotary_apply(const it_rotary* rotary, const void* x, int32_t dtype, int64_t token_stride,
                        const int32_t* positions, int32_t n_tokens, int32_t n_heads, int32_t head_dim,
                        int32_t transpose, void* out, int64_t out_stride, void* stream);
/* Rotation then append: rotated q to q_out, rotated k and v as it is into the
 * cache's pages in its format (each rounded or quantised once, from fp32).
 *   q: [n_tokens][n_heads][head_dim], k, v: [n_tokens][n_kv_heads][head_dim] of
 *     src_dtype F32, F16 or BF16, q_stride / k_stride / v_stride elements
 *     between tokens (a fused projection's rows: all three the same)
 *   n_heads: a multiple of n_kv_heads; 0: no q (q, q_out NULL)
 *   slot_mapping: int64[n_tokens] (slot < 0 = padding: q still rotated)
 *   positions: int32[n_tokens]; a negative one is latched
 *     (it_kv_cache_check) and its token writes nothing
 *   q_out: [n_tokens][n_heads][head_dim] contiguous, of q_out_dtype F32, F16 or
 *     BF16; may be q itself where that is contiguous and of that dtype */
int32_t it_kv_append_rotary(it_kv_cache* cache, const it_rotary* rotary, const void* q, const void* k,
                            const void* v, int32_t src_dtype, int64_t q_stride, int64_t k_stride,
                            int64_t v_stride, int32_t n_heads, const int64_t* slot_mapping,
                            const int32_t* positions, int32_t n_tokens, void* q_out, int32_t q_out_dtype,
                            void* stream);

/* Block-table gather: materialise the contiguous slices that
 * forward.rs:233-243 reads, through a block table.
 *   block_tables: int32[n_seqs][max_blocks] (absolute logical block index)
 *   ctx_lens: int32[n_seqs]; start_pos: int32[n_seqs] or NULL (all 0)
 *   cu_out: int64[n_seqs] output token offset of each sequence
 *   max_tokens: upper bound of ctx_lens[b] - start_pos[b] (sizes the grid)
 * Output for sequence b: [n_kv_heads][ctx_b - start_b][head_dim] at token
 * offset cu_out[b] (element offset cu_out[b]*n_kv_heads*head_dim).  A Q8_0
 * cache writes packed 34-byte BlockQ8_0 records, head_dim/32 per row; a Q4_0
 * cache 18-byte BlockQ4_0 records, a Q4_1 cache 20-byte BlockQ4_1 ones, Q5_0
 * and Q5_1 caches 22- and 24-byte ggml block_q5_0 / block_q5_1 records. */
int32_t it_kv_gather(const it_kv_cache* cache, const int32_t* block_tables, int32_t max_blocks,
                     const int32_t* ctx_lens, const int32_t* start_pos, const int64_t* cu_out,
                     int32_t n_seqs, int32_t max_tokens, void* k_out, void* v_out, void* stream);

/* Evict: zero every page (all heads, K and V, every layer) of the given
 * blocks, so a recycled block starts clean.  blocks: int32[n], device. */
int32_t it_kv_evict(it_kv_cache* cache, const int32_t* blocks, int32_t n, void* stream);

/* Keep a device block table in step with the slot mapping: for each token
 * i with slots[i] >= 0, tables[seq[i]][pos[i] / block_size] :=
 * slots[i] / block_size (every token of a block writes the same id).
 * tables: int32[n_seqs][max_blocks]; seq, pos: int32[n]; slots:
 * int64[n]; all device.  Out-of-range entries are skipped and latched
 * (it_kv_cache_check). */
int32_t it_kv_sync_tables(it_kv_cache* cache, int32_t* tables, int32_t max_blocks, int32_t n_seqs,
                          const int32_t* seq, const int32_t* pos, const int64_t* slots, int32_t n,
                          void* stream);

/* Copy-on-write page copy: block dst[i] := block src[i] (all heads, K, V,
 * every layer). */
int32_t it_kv_copy_blocks(it_kv_cache* cache, const int32_t* src, const int32_t* dst, int32_t n,
                          void* stream);

/* Move token rows between slots: for each i, in every layer and head, the K
 * and V row of slot src[i] becomes that of slot dst[i].  With `rotary`, K rows
 * are also turned by delta[i] positions (new position - old position; K is
 * cached rotated), without its magnitude, which they already carry: F32, F16
 * and BF16 rows are turned in fp32 and rounded once, quantised rows are
 * dequantised, turned and quantised again; a row with delta 0 keeps its bytes.
 *   src, dst: int64[n], device; a pair with a negative slot is skipped; slots
 *     out of range are latched and skipped
 *   rotary: NULL = copy as it is; delta: int32[n], device, NULL only without it
 * dst slots must be distinct and none may be another pair's src (fresh blocks,
 * as one call of it_kv_manager_compact or _compact_many hands out); src[i] == dst[i] is allowed: the row
 * is turned in place (a shift of a sequence's positions).  Takes a multi-layer
 * cache or a layer's view. */
int32_t it_kv_move(it_kv_cache* cache, const int64_t* src, const int64_t* dst, int32_t n,
                   const it_rotary* rotary, const int32_t* delta, void* stream);

/* ======================================================================== */
/* Device: attention over the cache.                                         */
/* ======================================================================== */
/* Workspace bytes it_paged_decode needs (fp32 partial (m, l, O) for every
 * (sequence, head, partition)). */
size_t it_paged_decode_workspace(int32_t n_seqs, int32_t n_heads, int32_t head_dim,
                                 int32_t max_tokens, int32_t partition);

/* Partition (tokens per split) for it_paged_decode over contexts the caller
 * knows on the host, as a batcher does: the smallest multiple of 64 in
 * [64, 2048] whose non-empty (sequence, KV head, partition) units run in the
 * fewest rounds of four resident workgroups per compute unit.  Short
 * partitions keep each workgroup's chain of dependent page loads short;
 * units beyond the resident slots would run a second round.  A batch that
 * needs more than two rounds at any size takes the longest partition that
 * keeps two workgroups per compute unit instead (fewest partials).
 * Quantised caches at head_dim 128 run up to eight workgroups per unit (six
 * for some head counts): where four would take partitions above 384 tokens, the
 * same is planned over the partitions that leave room for all of them (or
 * seven), and the longest is that which leaves room for all.
 *   ctx_lens, start_pos: host int32[n_seqs] (start_pos may be NULL)
 *   n_cu: compute units of the device (0 = ask the current HIP device)
 * No counterpart in the reference: flash_attn_f32 (flash_attn.rs:6-72) does
 * not split keys.  Its caller is the batcher's step (continuous.rs:28-74),
 * which holds the lengths. */
int32_t it_paged_decode_partition(int32_t dtype, int32_t head_dim, int32_t block_size, int32_t n_heads,
                                  int32_t n_kv_heads, const int32_t* ctx_lens, const int32_t* start_pos,
                                  int32_t n_seqs, int32_t n_cu, int32_t* partition);

/* Paged split-K flash-decode, one query per sequence.  For each sequence b
 * and query head h the result equals flash_attn_f32 (flash_attn.rs:6-72)
 * over keys start_b..ctx_b-1 of KV head h*Hkv/Hq (forward.rs:231-254),
 * within fp32 tolerance.
 *   q: [n_seqs][n_heads][head_dim]; q_dtype F32 (F32 and quantised caches),
 *      BF16 (BF16 cache) or F16 (F16 cache); 16-byte aligned
 *   block_tables/ctx_lens/start_pos: as it_kv_gather
 *   max_tokens: upper bound of ctx_b - start_b
 *   partition: tokens per split, a multiple of 64 in [64, 2048]
 *              (it_paged_decode_partition picks one for a batch)
 *   ws: it_paged_decode_workspace(...) bytes, device, 256-byte aligned
 *   out: [n_seqs][n_heads][head_dim] of out_dtype (F32 or q_dtype); 8-byte
 *        aligned for F32, 4-byte for 16-bit types
 * Two kernels: the split pass writes (m, l, O) per partition, the combine
 * pass merges them.  n_heads must be a multiple of n_kv_heads. */
int32_t it_paged_decode(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                        const int32_t* block_tables, int32_t max_blocks, const int32_t* ctx_lens,
                        const int32_t* start_pos, int32_t n_seqs, int32_t max_tokens, float scale,
                        int32_t partition, void* ws, size_t ws_bytes, void* out,
                        int32_t out_dtype, void* stream);

/* The two passes of it_paged_decode as separate launches, same arguments:
 * it_paged_decode_split then it_paged_decode_combine on one stream equals
 * it_paged_decode (lets a caller time or schedule the passes apart). */
int32_t it_paged_decode_split(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                              const int32_t* block_tables, int32_t max_blocks, const int32_t* ctx_lens,
                              const int32_t* start_pos, int32_t n_seqs, int32_t max_tokens, float scale,
                              int32_t partition, void* ws, size_t ws_bytes, void* out, int32_t out_dtype,
                              void* stream);
int32_t it_paged_decode_combine(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                                const int32_t* block_tables, int32_t max_blocks, const int32_t* ctx_lens,
                                const int32_t* start_pos, int32_t n_seqs, int32_t max_tokens, float scale,
                                int32_t partition, void* ws, size_t ws_bytes, void* out, int32_t out_dtype,
                                void* stream);

/* it_paged_decode without a workspace argument.  No counterpart in the
 * reference: it is for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  The
 * partials live in a 32 MiB device array of the library (one per GPU, held
 * until the process ends); a call that needs more than that
 * (it_paged_decode_workspace > 32 MiB) is IT_INVALID_INPUT.  It allocates
 * nothing: the array's device address is looked up once per device, on the
 * first call there.  Calls on one GPU share the array, so calls that
 * overlap in time on one GPU (different streams) race.  Other arguments and
 * results as it_paged_decode. */
int32_t it_paged_decode_noalloc(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                                const int32_t* block_tables, int32_t max_blocks, const int32_t* ctx_lens,
                                const int32_t* start_pos, int32_t n_seqs, int32_t max_tokens, float scale,
                                int32_t partition, void* out, int32_t out_dtype, void* stream);

/* Chunked prefill attention over the cache (the chunk's K/V already
 * appended).  Sequence b has q_len_b = cu_q[b+1]-cu_q[b] query rows at
 * positions ctx_b - q_len_b + i; with causal != 0 row i attends keys
 * 0..ctx_b - q_len_b + i, else all ctx_b keys.
 *   q/out: [cu_q[n_seqs]][n_heads][head_dim], BF16 q; out F32 or BF16
 *   cu_q: int32[n_seqs+1], device; max_q_len bounds q_len_b. */
int32_t it_paged_prefill(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                         const int32_t* cu_q, int32_t max_q_len, const int32_t* block_tables,
                         int32_t max_blocks, const int32_t* ctx_lens, int32_t n_seqs, float scale,
                         int32_t causal, void* out, int32_t out_dtype, void* stream);
/* Bytes of device workspace with which it_paged_prefill_ws can cut a call's
 * work over the keys; 0 if it would not (a launch of this size fills the
 * device without).  Bounded: at most 70 MB.  max_blocks x block_size bounds the
 * contexts: a caller that knows the longest asks with its blocks instead of the
 * table's width, and passes no workspace where the answer is 0 (then the call
 * is one launch).  Where a workspace is passed it is of the table's width. */
size_t it_paged_prefill_workspace(int32_t n_heads, int32_t n_kv_heads, int32_t n_seqs, int32_t max_q_len,
                                  int32_t max_blocks, int32_t block_size);
/* it_paged_prefill with a workspace (device, 256-byte aligned,
 * it_paged_prefill_workspace(...) bytes; NULL = none).  When the sequences'
 * lengths leave the device with few workgroups (a chunk of one long
 * context), the keys of each query block are divided among several, whose
 * fp32 partial (m, l, O) go through the workspace to a second kernel that
 * merges them.  The number of divisions follows from all sequences of the call
 * and from max_blocks, so a row's result may differ between batches, and
 * between calls with and without a workspace, by the rounding of its
 * probabilities to 16 bits against other maxima; without one it depends on the
 * row's own sequence alone. */
int32_t it_paged_prefill_ws(const it_kv_cache* cache, const void* q, int32_t q_dtype, int32_t n_heads,
                            const int32_t* cu_q, int32_t max_q_len, const int32_t* block_tables,
                            int32_t max_blocks, const int32_t* ctx_lens, int32_t n_seqs, float scale,
                            int32_t causal, void* ws, size_t ws_bytes, void* out, int32_t out_dtype,
                            void* stream);

/* CoreOperator::FlashAttention as ArmCpuBackend executes it
 * (src/backend/arm.rs:304-370): every one of n_heads query heads attends
 * the same K/V [n_kv][head_dim] with scale 1/sqrtf(head_dim) and an
 * optional additive mask [n_kv] (NULL = none; -inf skips the key).
 *   q/out: [n_heads][head_dim] F32; k, v: [n_kv][head_dim] F32; device.
 *   ws: it_flash_attention_workspace(...) bytes, device. */
size_t it_flash_attention_workspace(int32_t n_heads, int32_t head_dim, int32_t n_kv);
int32_t it_flash_attention(const float* q, const float* k, const float* v, const float* mask,
                           float* out, int32_t n_heads, int32_t head_dim, int32_t n_kv, void* ws,
                           size_t ws_bytes, void* stream);

/* ======================================================================== */
/* Device: the next token.  The reference's step ends with                  */
/* ForwardExecutor::sample (src/inference/forward.rs:765-796); a batcher's   */
/* rows each have settings of their own.                                     */
/* ======================================================================== */
/* One token per row of logits z from a given uniform number u:
 *   order: z descending, equal z by the lower token first; NaN counts as -inf,
 *     tokens at -inf are never drawn
 *   w_i = exp((z_i - max z) / temperature)  (a maximum of +inf: the tokens at
 *     +inf weigh 1, all others nothing)
 *   min-p keeps w_i >= min_p (the largest weight is 1); then top-k the first k;
 *     then top-p those whose mass before them is below top_p of the mass left;
 *     the first of the order is always kept
 *   token = the first kept one with cumulative mass > u * kept mass
 *   prob = its share of the kept mass
 * temperature <= 0 (or NaN): the first of the order, prob 1.  A row with
 * nothing above -inf: token -1, prob 0.
 * Masses are 64-bit integers in units of 2^-44 of the largest token's, each
 * rounded to nearest once: sums are exact, so a result depends on neither the
 * batch nor the order of the sums.
 *   logits: [n_rows][vocab] of F32, F16 or BF16, row_stride elements between
 *     rows; n_rows 0 .. 65535, vocab 1 .. 262144
 *   u: float[n_rows], device, in [0, 1) (below 0 and NaN count as 0, 1 and
 *     above as the last kept token)
 *   temperatures, top_ps, min_ps: float[n_rows], top_ks: int32[n_rows], device;
 *     NULL: temperature / top_k / top_p / min_p holds for every row (finite,
 *     temperature >= 0, min_p <= 1).  Off: top_k <= 0, top_p >= 1, min_p <= 0;
 *     min_p above 1 counts as 1, NaN as off
 *   tokens: int32[n_rows]; probs: float[n_rows] or NULL; device
 *   ws: it_sample_workspace(...) bytes, device, 256-byte aligned; it need not
 *     be cleared, and calls that overlap in time need one each; short rows and
 *     large batches need none (0 bytes: ws may be NULL)
 * Launched on the current device, to which `stream` must belong. */
size_t it_sample_workspace(int32_t n_rows, int32_t vocab);
int32_t it_sample(const void* logits, int32_t dtype, int64_t row_stride, int32_t n_rows, int32_t vocab,
                  const float* u, const float* temperatures, const int32_t* top_ks, const float* top_ps,
                  const float* min_ps, float temperature, int32_t top_k, float top_p, float min_p,
                  int32_t* tokens, float* probs, void* ws, size_t ws_bytes, void* stream);

/* ======================================================================== */
/* Device: latent attention.  Keys and values of all heads come from one     */
/* shared row a token, [c | r]: a latent c of latent_dim elements, from which */
/* each head's key and value are projected, and a rotated key r of rope_dim   */
/* elements that all heads share.  Head h's score against token j is          */
/*   scale * (q_h . k_hj + qr_h . r_j),  k_hj = W_h c_j,  v_hj = U_h c_j.     */
/* Absorbed (it_latent_decode): (W_h^T q_h) . c_j, the cached rows read as    */
/* they are, once for all heads, and U_h applied to the result by the caller. */
/* Expanded (it_latent_prefill): k and v projected up by the caller.  No      */
/* counterpart in the reference, whose caches are per head (forward.rs:16-19).*/
/* ======================================================================== */
/* A cache of such rows: one pool, [n_layers][num_blocks] pages of block_size
 * rows of latent_dim + rope_dim elements of F32, F16 or BF16.  The pool is
 * it_kv_cache_desc's k_pool, head_dim a row's elements, n_kv_heads 1, v_pool
 * NULL.  it_kv_evict, it_kv_copy_blocks, it_kv_sync_tables, it_kv_cache_layer,
 * _describe, _check and _destroy take it as they take any cache; it_kv_gather
 * writes its rows to k_out (v_out NULL); it_kv_move turns the rope part alone
 * (rotary of rope_dim elements).  Entry points for K and V rows refuse it.
 * latent_dim 8 .. 1024, rope_dim 8 .. 256, both multiples of 8. */
int32_t it_kv_cache_new_latent(int32_t device, int32_t n_layers, int64_t num_blocks, int32_t block_size,
                               int32_t latent_dim, int32_t rope_dim, int32_t dtype, it_kv_cache** out);
/* Wraps a caller-owned pool of n_layers * num_blocks pages (16-byte aligned). */
int32_t it_kv_cache_wrap_latent(int32_t device, int32_t n_layers, void* pool, int64_t num_blocks,
                                int32_t block_size, int32_t latent_dim, int32_t rope_dim, int32_t dtype,
                                it_kv_cache** out);
/* latent_dim of a latent cache, 0 of any other (and of NULL). */
int32_t it_kv_cache_latent_dim(const it_kv_cache* cache);

/* Latent rows into the cache, and the rope part of the queries beside them:
 *   c' = c * rsqrt(mean(c^2) + eps) * weight  (weight NULL: c as it is)
 *   r' = R(position) r,  q' = R(position) q    (rotary NULL: as they are)
 * in fp32, each result rounded once.
 *   kv: [n_tokens][latent_dim + rope_dim] of src_dtype F32, F16 or BF16,
 *     kv_stride elements between tokens (the down projection's rows)
 *   weight: [latent_dim] of weight_dtype F32, F16 or BF16
 *   q: [n_tokens][n_heads][rope_dim] of src_dtype, q_stride elements between
 *     tokens, q_head_stride between heads (the rope part of a projection's
 *     heads); n_heads 0: none (q, q_out NULL).  q_out: the same shape, of
 *     q_out_dtype F32, F16 or BF16, with strides of its own; may be q itself
 *     (same strides and dtype)
 *   Otherwise q_out and rows_out lie on no other tensor; between its rows they
 *     may, where both are equally many bytes apart from token to token (q, q_out
 *     and kv as parts of one projection)
 *   rows_out: NULL, or [n_tokens][latent_dim + rope_dim] of the cache's dtype,
 *     contiguous: the stored rows, padding tokens' too (what a prompt's
 *     projection up reads)
 *   slot_mapping: int64[n_tokens] (slot < 0 = padding: nothing is stored)
 *   positions: int32[n_tokens], NULL without rotary; a negative one is latched
 *     (it_kv_cache_check) and its token writes nothing
 *   rotary: n_dims = rope_dim */
int32_t it_latent_append(it_kv_cache* cache, const it_rotary* rotary, const void* kv, int32_t src_dtype,
                         int64_t kv_stride, const void* weight, int32_t weight_dtype, float eps, const void* q,
                         int64_t q_stride, int64_t q_head_stride, int32_t n_heads, void* q_out,
                         int32_t q_out_dtype, int64_t out_stride, int64_t out_head_stride, void* rows_out,
                         const int64_t* slot_mapping, const int32_t* positions, int32_t n_tokens, void* stream);

/* Absorbed latent attention over the cache: q_len new tokens of each sequence
 * (their rows already appended), the last of its context.  For head h of the
 * sequence's new token i (position p = ctx - q_len + i)
 *   out = sum_j softmax_j(scale (q_latent . c_j + q_rope . r_j)) c_j
 * over the cached tokens start .. p; a row that sees none is 0.
 *   q_latent: [n_seqs * q_len][n_heads][latent_dim], q_rope: [..][rope_dim],
 *     each with element strides between tokens and heads (parts of one tensor
 *     too), of q_dtype: the cache's dtype
 *   n_heads 1 .. 1024, q_len 1 .. 64; block_tables, ctx_lens, start_pos: as
 *     it_kv_gather
 *   max_tokens: upper bound of ctx_b - floor32(start_b) (a longer sequence is
 *     latched and gives 0, as does one with a negative start)
 *   ws: it_latent_decode_workspace(...) bytes of device memory, 256-byte
 *     aligned, for the partial results of sequences that several workgroups
 *     share; calls that overlap in time need one each
 *   out: [n_seqs * q_len][n_heads][latent_dim] of out_dtype: F32 or q_dtype,
 *     16-byte aligned, apart from the inputs
 *   n_seqs * max_tokens (or what max_blocks hold) at most about 2^35
 * Sums and the softmax in fp32; for F16 and BF16 caches the probabilities are
 * rounded to the cache's type for the matrix cores.  How the keys are divided
 * follows from all sequences of the call, so a row's result may differ between
 * batches by that rounding. */
size_t it_latent_decode_workspace(const it_kv_cache* cache, int32_t n_seqs, int32_t q_len, int32_t n_heads,
                                  int32_t max_tokens);
int32_t it_latent_decode(const it_kv_cache* cache, const void* q_latent, const void* q_rope, int32_t q_dtype,
                         int64_t ql_stride, int64_t ql_head_stride, int64_t qr_stride, int64_t qr_head_stride,
                         int32_t n_heads, int32_t q_len, const int32_t* block_tables, int32_t max_blocks,
                         const int32_t* ctx_lens, const int32_t* start_pos, int32_t n_seqs, int32_t max_tokens,
                         float scale, void* ws, size_t ws_bytes, void* out, int32_t out_dtype, void* stream);

/* Expanded latent attention over contiguous keys and values: per head a key
 * part and a value projected from the latents, and one rope key for all heads.
 *   q: [total_q][n_heads][nope_dim + rope_dim], k: [total_k][n_heads][nope_dim],
 *   v: [total_k][n_heads][v_dim], k_rope: [total_k][rope_dim] of dtype F32, F16
 *     or BF16; element strides between tokens and heads (k and v may be parts
 *     of one projection, k_rope a part of the gathered rows)
 *   cu_q, cu_k: int32[n_seqs + 1], device: rows of each sequence, 0 first; with
 *     causal != 0 query i of a sequence sees its keys 0 .. k_len - q_len + i,
 *     else all k_len; a query that sees none is 0.  An infinite value is in the
 *     sums of the queries that see it: infinite, or NaN beside one of the other
 *     sign, or where its weight is 0 (F16, BF16: rounds to 0)
 *   max_q_len, max_k_len: upper bounds; a sequence past them, or outside
 *     total_q / total_k, is not computed and its rows are left as they are, as
 *     are rows behind the last sequence
 *   nope_dim, rope_dim, v_dim: multiples of 8, nope_dim + rope_dim <= 1024,
 *     v_dim <= 1024; fastest: F16 and BF16 with nope_dim and v_dim 64 or 128,
 *     rope_dim 32 or 64, and 16-byte aligned rows
 *   out: [total_q][n_heads][v_dim] contiguous, of out_dtype F32 or dtype,
 *     16-byte aligned, apart from the inputs
 * Launched on the current device, to which `stream` must belong. */
int32_t it_latent_prefill(const void* q, const void* k, const void* v, const void* k_rope, int32_t dtype,
                          int64_t q_stride, int64_t q_head_stride, int64_t k_stride, int64_t k_head_stride,
                          int64_t v_stride, int64_t v_head_stride, int64_t rope_stride, int32_t n_heads,
                          int32_t nope_dim, int32_t rope_dim, int32_t v_dim, const int32_t* cu_q,
                          const int32_t* cu_k, int32_t n_seqs, int32_t total_q, int32_t total_k,
                          int32_t max_q_len, int32_t max_k_len, float scale, int32_t causal, void* out,
                          int32_t out_dtype, void* stream);

/* ======================================================================== */
/* Device: beam search.  The reference draws one token a step                */
/* (src/inference/forward.rs:765-796) and carries one hypothesis.            */
/* ======================================================================== */
/* The best continuations of each group's beams.  Candidate (b, i), beam b of
 * the group and token i, has the value
 *   v = scores[b] + log_softmax(z_b)_i
 *     = (scores[b] - log sum_j exp(z_bj - m_b)) + (z_bi - m_b), m_b = max_j z_bj
 * in fp64, and candidates are ordered by v descending, equal v by the lower
 * beam, then the larger logit (far enough below the row's maximum, v does not
 * tell logits apart), then the lower token.  NaN logits and scores count as -inf; a candidate at -inf is
 * none; a row whose maximum is +inf weighs its tokens at +inf alone, equally.
 *   logits: [n_groups * n_beams][vocab] of F32, F16 or BF16, row_stride
 *     elements between rows; n_beams 1 .. 64, vocab 1 .. 262144
 *   scores: float[n_groups][n_beams], the beams' log-probabilities so far
 *     (-inf: the beam is not in use)
 *   n_out: 1 .. 64 (twice n_beams leaves n_beams of them beside those that end)
 *   out_scores: float[n_groups][n_out], v rounded; parents: int32 (the beam in
 *     its group) and tokens: int32 likewise.  Places without a candidate:
 *     -inf, -1, -1
 *   ws: it_beam_select_workspace(...) bytes, device, 256-byte aligned; it need
 *     not be cleared, and calls that overlap in time need one each
 * A result depends on neither the other groups nor the order of the sums.
 * Launched on the current device, to which `stream` must belong. */
size_t it_beam_select_workspace(int32_t n_groups, int32_t n_beams, int32_t vocab, int32_t n_out);
int32_t it_beam_select(const void* logits, int32_t dtype, int64_t row_stride, int32_t n_groups, int32_t n_beams,
                       int32_t vocab, const float* scores, int32_t n_out, float* out_scores, int32_t* parents,
                       int32_t* tokens, void* ws, size_t ws_bytes, void* stream);
/* Per-beam states put in a new order, in place: in each of n_outer arrays
 * (outer_stride bytes apart), row g * n_beams + j becomes what row
 * g * n_beams + parents[g][j] was (parents below 0 or not below n_beams: it
 * stays).  Block tables, token histories, recurrent states of every layer.
 *   x: rows of row_bytes bytes, row_stride bytes apart; n_beams 1 .. 64
 *   parents: int32[n_groups][n_beams], device, not inside x
 * Rows of 16-byte multiples at aligned addresses run fastest.  Launched on the
 * current device, to which `stream` must belong. */
int32_t it_beam_reorder(void* x, int64_t row_bytes, int64_t row_stride, int32_t n_outer, int64_t outer_stride,
                        int32_t n_groups, int32_t n_beams, const int32_t* parents, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* IT_KV_H */
