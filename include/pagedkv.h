/*
 * pagedkv.h -- C ABI of the MI355X paged-KV engine (libpagedkv.so).
 *
 * This is the drop-in boundary under the candle provider's `engine = "paged"`
 * path of einyx/ai-engine.  Every entry point is plain C: opaque handles,
 * raw pointers, sizes and an int status.  No torch, HIP or Rust types cross
 * it; HIP streams are passed as `void*` (a hipStream_t, NULL = default stream).
 *
 * Reference interfaces replaced (paths relative to the reference repository):
 *   KvPool::new            crates/ai-engine-candle/src/paged/attention.rs:39-55
 *   KvPool::write          crates/ai-engine-candle/src/paged/attention.rs:57-83
 *   KvPool::gather_seq     crates/ai-engine-candle/src/paged/attention.rs:85-97
 *   build_mask + sdpa      crates/ai-engine-candle/src/paged/attention.rs:11-28,100-136
 *   decode attention slice crates/ai-engine-candle/src/paged/transformer.rs:271-292
 *   prefill attention      crates/ai-engine-candle/src/paged/transformer.rs:139-196
 *   BlockAllocator/Table   crates/ai-engine-candle/src/paged/block_table.rs:5-58
 *
 * Conventions shared by every call:
 *  - Status: 0 = PKV_OK, negative = error.  The message of the last error of a
 *    pool is returned by pkv_last_error(pool); errors of calls that have no pool
 *    (create, allocator) by pkv_last_error(NULL) on the calling thread.
 *    No call unwinds, aborts or panics across the boundary.
 *  - Threading: a pool handle is externally synchronised (one caller thread at a
 *    time, like the reference's single engine thread, engine.rs:49).  Device
 *    work is enqueued on the caller's stream and is stream-ordered; the library
 *    starts no threads.
 *  - Pool layout (per layer, K and V separately), identical to the reference's
 *    KvPool tensors: [num_blocks][block_size][n_kv_head][head_dim], row-major,
 *    element type `dtype`.  Slot s = block_id * block_size + pos % block_size
 *    addresses the row [s][n_kv_head][head_dim] (attention.rs:88-91).
 *  - Device arrays (q, k, v, out, slot mappings, block tables, lengths) are
 *    device pointers unless the parameter name ends in `_host`.
 */
#ifndef PAGEDKV_H
#define PAGEDKV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define PKV_OK 0
#define PKV_ERR_INVALID (-1)     /* invalid argument or shape               */
#define PKV_ERR_OOM (-2)         /* device or host allocation failed        */
#define PKV_ERR_HIP (-3)         /* HIP runtime error                       */
#define PKV_ERR_UNSUPPORTED (-4) /* shape/dtype combination not provided    */
#define PKV_ERR_CAPACITY (-5)    /* allocator: free list too short          */
#define PKV_ERR_DEVICE_DATA (-6) /* kernel saw an out-of-range id/length    */

/* ---- element types ----------------------------------------------------- */
#define PKV_F32 0
#define PKV_F16 1
#define PKV_BF16 2
#define PKV_Q4 3 /* of pools only: 4 bits an element and 8 for a group's scale and offset */

/* ---- pool selectors ---------------------------------------------------- */
#define PKV_K 0
#define PKV_V 1

typedef struct pkv_pool pkv_pool;

/* Library version string, e.g. "pagedkv 0.1 gfx950". */
const char* pkv_version(void);

/* Message of the last failed call on `pool` (or of the calling thread when
 * pool is NULL).  Never NULL; "" when there was no error. */
const char* pkv_last_error(const pkv_pool* pool);

/* Allocate K and V pools for `n_layers` layers on HIP device `device`, zero
 * filled like Tensor::zeros in KvPool::new (attention.rs:39-55).  One handle
 * stands for the reference's Vec<KvPool> (engine.rs:70-72): layer l of the
 * handle is the reference's kv[l].  Block ids are shared by all layers.
 * dtype: PKV_F32 (the reference's own dtype), PKV_F16, PKV_BF16, or PKV_Q4
 * (no reference counterpart; see "a cache held in 4 bits").
 * Shape limits (PKV_ERR_UNSUPPORTED otherwise), narrower than the
 * reference's KvPool::new, which takes any sizes:
 *  - head_dim 64, 128 or 256.  The reference reads it from GGUF
 *    (`attention.key_length`, else embedding_length / head_count,
 *    arch.rs:77-83); every llama / qwen2 / qwen3 model of the supported
 *    architectures (arch.rs:27-36) has 64 or 128.
 *  - block_size a power of two in [1, 256].  The reference takes any
 *    usize (block_table.rs:17-30); its engine default and the block size of
 *    its tests is 16 (app.rs:701, tests/paged_parity.rs:33).  Sizes below
 *    16 run kernels that read a block id per lane (a 16-token attention
 *    tile then spans several blocks); other sizes (24, 48, ...) are
 *    refused: every kernel addresses a token's slot with shifts and masks.
 * n_kv_head is any count in 1 .. 1024, and the slab (2 * n_layers *
 * num_blocks * block_size * n_kv_head * head_dim elements) below 2^63
 * bytes (else PKV_ERR_UNSUPPORTED); the GQA ratio n_head / n_kv_head of the
 * attention calls is any positive integer (repeat_kv, attention.rs:113,
 * 128-136).  The pool is plain device memory from hipMalloc, allocated by
 * the library itself.  No kernel loads pool bytes that the same launch
 * stored (the fused appends hand the new rows to the attention through
 * LDS; a launch's copies and moves read each block before any write to it,
 * in the same thread), so results do not depend on the pool's caching
 * or coherence attributes. */
int pkv_pool_create(pkv_pool** out, int n_layers, int num_blocks,
                    int block_size, int n_kv_head, int head_dim, int dtype,
                    int device);
int pkv_pool_destroy(pkv_pool* pool);

/* Shape and placement queries. */
int pkv_pool_shape(const pkv_pool* pool, int* n_layers, int* num_blocks,
                   int* block_size, int* n_kv_head, int* head_dim, int* dtype);
size_t pkv_pool_layer_bytes(const pkv_pool* pool); /* bytes of one K (or V) */
int pkv_pool_layer_ptrs(const pkv_pool* pool, int layer, void** k, void** v);

/* Synchronous host<->pool byte copies (tests, debugging, checkpoints). */
int pkv_pool_read(pkv_pool* pool, int layer, int which, size_t byte_offset,
                  size_t nbytes, void* host_dst);
int pkv_pool_write(pkv_pool* pool, int layer, int which, size_t byte_offset,
                   const void* host_src, size_t nbytes);

/* Fill every layer's K and V with N(0,1) samples rounded to the pool dtype,
 * from a counter-based hash of (seed, layer, which, element index).
 * A workload generator for benchmarks; no reference counterpart. */
int pkv_pool_fill_normal(pkv_pool* pool, uint64_t seed, void* stream);

/* The check of pkv_pool_fill_normal after blocks have moved (copy-on-write,
 * compaction; no reference counterpart): counts, into *mismatches, the
 * 16-byte chunks of block blocks[i], over every layer's K and V, that differ
 * from what pkv_pool_fill_normal(seed) wrote into block origin[i].
 * blocks, origin: device int32 [n]; an id out of range counts the item as
 * mismatching and is reported by pkv_pool_check().  Synchronous. */
int pkv_pool_verify_normal(pkv_pool* pool, uint64_t seed, const int32_t* blocks,
                           const int32_t* origin, int n, uint64_t* mismatches,
                           void* stream);

/* Read every byte of blocks[i] in every layer's K and V and add their
 * 32-bit words (mod 2^64) into *sum, a device uint64 the caller zeroes;
 * asynchronous on `stream`.  No reference counterpart: the read rate of a
 * random block set (the decode roofline's read ceiling, bytes read / time)
 * and a checksum of the blocks.  blocks: device int32 [n]; an id out of
 * range is skipped and reported by pkv_pool_check(). */
int pkv_pool_read_blocks(pkv_pool* pool, const int32_t* blocks, int n, uint64_t* sum,
                         void* stream);

/* ---- KV append / scatter (KvPool::write, attention.rs:57-83) -----------
 * k, v: [n_tokens][n_kv_head][head_dim] in the pool dtype.
 * slot_mapping: [n_tokens] int32, slot = block * block_size + offset
 * (the host computes it with BlockAllocator::locate, block_table.rs:55-58).
 * Token i is copied bit-exactly to row slot_mapping[i] of layer `layer`'s K
 * and V pools; no other byte changes.  A negative slot skips the token
 * (padding); a slot >= num_blocks*block_size is not written and makes the
 * next pkv_pool_check() report PKV_ERR_DEVICE_DATA. */
int pkv_append(pkv_pool* pool, int layer, const void* k, const void* v,
               const int32_t* slot_mapping, int n_tokens, void* stream);

/* ---- gather (KvPool::gather_seq, attention.rs:85-97) -------------------
 * out_k, out_v: [len][n_kv_head][head_dim] pool dtype, bit-exact copies of
 * the rows at slot blocks[p / bs] * bs + p % bs, p = 0..len-1.
 * block_table: device int32 [ceil(len / block_size)]. */
int pkv_gather_seq(pkv_pool* pool, int layer, const int32_t* block_table,
                   int len, void* out_k, void* out_v, void* stream);

/* ---- gather of several sequences in one launch (no reference counterpart:
 * the batched form of gather_seq for callers that want the K/V of many
 * sequences contiguous, e.g. a varlen attention kernel) ------------------
 * Sequence b's positions 0 .. cu_lens[b+1]-cu_lens[b]-1 are copied, bit for
 * bit as by pkv_gather_seq with block_tables[b], to rows cu_lens[b] ..
 * cu_lens[b+1]-1 of out_k / out_v ([total_rows][n_kv_head][head_dim]).
 * cu_lens: device int32 [batch+1], cu_lens[0] = 0, nondecreasing;
 * total_rows = cu_lens[batch] (host value).  block_tables: device int32
 * [batch][max_blocks_per_seq].  batch <= 4096.  A block id out of range, or
 * a length beyond the table, zeroes those rows and is reported by
 * pkv_pool_check(). */
int pkv_gather_varlen(pkv_pool* pool, int layer, const int32_t* block_tables,
                      int max_blocks_per_seq, const int32_t* cu_lens, int batch,
                      int total_rows, void* out_k, void* out_v, void* stream);

/* ---- block copy (copy-on-write after fork; no reference counterpart) ----
 * For every layer and both K and V: block dst[i] <- block src[i], i < n.
 * src, dst: device int32 [n].  dst ids must be distinct and no dst may be a
 * src of the same call (the CoW contract: dst blocks are fresh); otherwise
 * the copies race.  An id out of range is skipped and reported by
 * pkv_pool_check().  With PKV_DEBUG set in the environment (to anything but
 * "0") the call first checks the contract on host copies of src and dst
 * (synchronising the stream) and returns PKV_ERR_INVALID, copying nothing,
 * if it is broken. */
int pkv_copy_blocks(pkv_pool* pool, const int32_t* src, const int32_t* dst,
                    int n, void* stream);

/* ---- compaction (no reference counterpart) ------------------------------
 * Moves block src_host[i] to dst_host[i] for every layer and K/V, in place:
 * the dst set may overlap the src set (e.g. survivors gathered into a
 * contiguous prefix).  src ids distinct, dst ids distinct.  The plan (chains
 * and cycles of the move graph) is built on the host, so ids are host arrays;
 * it is uploaded to a device buffer the pool allocates once, at creation,
 * for the largest plan.  Stream-ordered: the call returns once the moves are
 * enqueued (it waits only, if at all, for the previous call's plan upload
 * before reusing the pinned staging copy).  Each byte is read once and
 * written once; no scratch pool is allocated. */
int pkv_compact(pkv_pool* pool, const int32_t* src_host,
                const int32_t* dst_host, int n, void* stream);

/* ---- paged decode attention (sdpa + build_mask + the decode-step
 * attention slice, attention.rs:100-136, transformer.rs:271-292) ----------
 * One query token per sequence.
 *  q:            [batch][n_head][head_dim], pool dtype (post-RoPE).
 *  out:          [batch][n_head * head_dim], out_dtype (PKV_F32 or the pool
 *                dtype); element [b][h*head_dim + d] as in attention.rs:124-125.
 *  block_tables: [batch][max_blocks_per_seq] int32.
 *  context_lens: [batch] int32 = number of keys attended = seq_lens[b] + 1
 *                (the reference's valid_lens, transformer.rs:289).
 *  max_context_len: host int >= every context_lens[b] (the reference's
 *                kv_len, transformer.rs:241); sizes the partition grid.
 *                1 .. 2^30, and batch * n_kv_head * max(16, ceil(
 *                max_context_len / 1024)) below 2^26 (one 64-lane wave
 *                each; else PKV_ERR_INVALID / _UNSUPPORTED).
 *  scale:        multiplies q.k (the reference uses 1/sqrt(head_dim),
 *                attention.rs:118-120).
 *  k_new, v_new: NULL, or [batch][n_kv_head][head_dim]: then the call first
 *                stores them at token position context_lens[b]-1 of sequence
 *                b (KvPool::write at seq_lens[b], transformer.rs:276) and the
 *                attention sees them -- append and attention in one launch.
 * GQA: query head h reads kv head h / (n_head / n_kv_head) (attention.rs:128-136),
 * for any integer ratio; ratios above 16 run as one launch (and merge) per
 * slice of 16 query heads, each reading the group's K/V.
 * fp32 accumulation; softmax in fp32 with an exp2 formulation.
 * context_lens[b] == 0 yields a zero output row.
 * Mask: key k of row b is attended iff k < context_lens[b] -- the
 * reference's build_mask(seq_lens + 1, positions, kv_len) as the decode step
 * calls it, where positions == seq_lens (transformer.rs:289-290,
 * engine.rs:130-133), so its second bound k <= positions[b]
 * (attention.rs:22) coincides with the first.  Callers whose positions
 * differ from seq_lens use pkv_decode_attention_positions. */
int pkv_decode_attention(pkv_pool* pool, int layer, const void* q, void* out,
                         int out_dtype, const int32_t* block_tables,
                         int max_blocks_per_seq, const int32_t* context_lens,
                         int max_context_len, int batch, int n_head,
                         float scale, const void* k_new, const void* v_new,
                         void* stream);

/* pkv_decode_attention with build_mask's second bound (attention.rs:11-28):
 * key k of row b is attended iff k < context_lens[b] and k <= positions[b],
 * positions being the rows' query positions (the reference's q_positions,
 * transformer.rs:290).  positions: device int32 [batch], non-NULL.  k_new /
 * v_new are still stored at context_lens[b] - 1 (KvPool::write at seq_lens,
 * transformer.rs:276) and attended only when positions[b] >=
 * context_lens[b] - 1.  A negative position attends no key: the row is
 * zero, nothing is stored for it, and pkv_pool_check() reports
 * PKV_ERR_DEVICE_DATA.  Other arguments and limits as pkv_decode_attention;
 * the split-context merge uses the same bounded lengths. */
int pkv_decode_attention_positions(pkv_pool* pool, int layer, const void* q, void* out,
                                   int out_dtype, const int32_t* block_tables,
                                   int max_blocks_per_seq, const int32_t* context_lens,
                                   const int32_t* positions, int max_context_len, int batch,
                                   int n_head, float scale, const void* k_new, const void* v_new,
                                   void* stream);

/* Workspace that pkv_decode_attention needs for a given batch/length; the
 * pool grows its internal workspace on demand with a hipMalloc.  The buffer
 * it replaces stays allocated, since queued work may still read it, until
 * the next reserve call, pkv_pool_destroy, or a later growth that would
 * otherwise keep more retired bytes than the new workspace holds (that
 * growth synchronises the device and frees them).  Callers that must not
 * allocate or synchronise later (stream capture, serving loops) reserve the
 * largest shape they will use up front; the reserve calls synchronise the
 * device when they free replaced buffers. */
size_t pkv_decode_workspace_bytes(const pkv_pool* pool, int batch, int n_head,
                                  int max_context_len);
int pkv_pool_reserve_decode(pkv_pool* pool, int batch, int n_head,
                            int max_context_len);

/* pkv_decode_attention without any allocation.  No counterpart in the
 * reference: for callers that cannot allocate device memory during a call
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Same arguments, kernels and results as pkv_decode_attention
 * (bit for bit), but the split-context partials go to a static device array
 * of PKV_NOALLOC_SCRATCH_BYTES that every GPU the library runs on holds for
 * the life of the process, not to the pool's workspace; the call makes no
 * hipMalloc, hipFree or other allocating call and records no profile
 * events.  A launch whose partials need more than the array
 * (pkv_decode_workspace_bytes > PKV_NOALLOC_SCRATCH_BYTES, e.g. batch 256
 * with contexts up to 32k on 8 kv heads of 128) returns PKV_ERR_UNSUPPORTED
 * before anything is enqueued.  All calls on one GPU share its array, so
 * calls that overlap on one GPU (different streams, threads or pools)
 * race: the caller orders them, e.g. on one stream. */
#define PKV_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
int pkv_decode_attention_noalloc(pkv_pool* pool, int layer, const void* q, void* out,
                                 int out_dtype, const int32_t* block_tables,
                                 int max_blocks_per_seq, const int32_t* context_lens,
                                 int max_context_len, int batch, int n_head,
                                 float scale, const void* k_new, const void* v_new,
                                 void* stream);

/* ---- chunked prefill attention (prefill_seq attention,
 * transformer.rs:139-196, generalised to a prior context) -----------------
 * Sequence s has q_len_s = cu_q_lens[s+1]-cu_q_lens[s] query tokens whose K/V
 * are already in the pool (pkv_append); its context has context_lens[s] keys
 * in total, so query i sits at position context_lens[s]-q_len_s+i and
 * attends keys 0..that position (causal; the reference's mask j > i -> -inf
 * when the prior context is empty).
 *  q:   [total_q][n_head][head_dim] pool dtype;  out: [total_q][n_head*head_dim].
 *  cu_q_lens: [n_seqs+1] int32; context_lens: [n_seqs] int32;
 *  block_tables: [n_seqs][max_blocks_per_seq] int32.
 *  max_q_len, max_context_len: host upper bounds, at most 2^30.  scale > 0 and finite
 *  (the reference's 1/sqrt(head_dim)); otherwise PKV_ERR_INVALID.
 *  Any GQA ratio n_head / n_kv_head; every pool dtype and head_dim. */
int pkv_prefill_attention(pkv_pool* pool, int layer, const void* q, void* out,
                          int out_dtype, const int32_t* cu_q_lens,
                          const int32_t* context_lens,
                          const int32_t* block_tables, int max_blocks_per_seq,
                          int n_seqs, int max_q_len, int max_context_len,
                          int n_head, float scale, void* stream);

/* pkv_prefill_attention with the chunk's K/V stored in the same launch (the
 * reference stores every prompt token with KvPool::write before attending,
 * transformer.rs:173-177; pkv_append + pkv_prefill_attention in one call).
 * k_new, v_new: [total_q][n_kv_head][head_dim] in the pool dtype, 16-byte
 * aligned; token i of sequence s is stored at its position
 * context_lens[s] - q_len_s + i (slot from block_tables) and attended from
 * these rows, so the result and the pool afterwards equal pkv_append
 * followed by pkv_prefill_attention.  A block id out of range is reported by
 * pkv_pool_check(). */
int pkv_prefill_attention_append(pkv_pool* pool, int layer, const void* q,
                                 void* out, int out_dtype,
                                 const int32_t* cu_q_lens,
                                 const int32_t* context_lens,
                                 const int32_t* block_tables,
                                 int max_blocks_per_seq, int n_seqs,
                                 int max_q_len, int max_context_len,
                                 int n_head, float scale, const void* k_new,
                                 const void* v_new, void* stream);

/* Workspace of pkv_prefill_attention for the given launch shape: launches
 * with few row blocks (fewer than can fill the GPU) split long key ranges
 * into parts that are merged afterwards, with partial results in the pool's
 * workspace (0: no split).  The pool grows the workspace on demand;
 * callers that must not allocate later reserve it up front. */
size_t pkv_prefill_workspace_bytes(const pkv_pool* pool, int n_seqs, int n_head,
                                   int max_q_len, int max_context_len);
int pkv_pool_reserve_prefill(pkv_pool* pool, int n_seqs, int n_head,
                             int max_q_len, int max_context_len);

/* ---- a layer's mixed batch in one call (engine step of run_loop,
 * engine.rs:62-237: some sequences prefill a prompt chunk, the others decode
 * one token; the reference attends them one sequence at a time,
 * transformer.rs:139-196 and 271-292) -------------------------------------
 * The arguments of pkv_prefill_attention(_append) and of
 * pkv_decode_attention, as two structs; n_head and scale are shared.  The
 * result (every output row, every stored K/V row, pkv_pool_check's error
 * bits) is identical, bit for bit, to pkv_prefill_attention(_append)
 * followed by pkv_decode_attention on the same stream: for 16-bit pools with
 * head_dim 64 or 128 and n_head / n_kv_head of 4 or 8 (f16 at head_dim 128:
 * 8 only) both run in one kernel launch, their workgroups sharing the CUs
 * (the prefill is bound by MFMA and instruction issue, the decode by HBM);
 * other shapes run the two calls in sequence.  A NULL batch, or one with
 * n_seqs / batch == 0, leaves just the other call.  The two batches must
 * not share the blocks their new rows are stored in (under copy-on-write a
 * sequence appends only to blocks it alone holds).  Workspace: the decode
 * partials and the prefill split partials side by side
 * (pkv_mixed_workspace_bytes). */
typedef struct pkv_prefill_batch {
  const void* q;               /* [total_q][n_head][head_dim], pool dtype */
  void* out;                   /* [total_q][n_head * head_dim], out_dtype */
  int out_dtype;
  const int32_t* cu_q_lens;    /* [n_seqs + 1] */
  const int32_t* context_lens; /* [n_seqs] */
  const int32_t* block_tables; /* [n_seqs][max_blocks_per_seq] */
  int max_blocks_per_seq;
  int n_seqs;
  int max_q_len;
  int max_context_len;
  const void* k_new;           /* chunk K/V stored by the call, or both NULL */
  const void* v_new;
} pkv_prefill_batch;

typedef struct pkv_decode_batch {
  const void* q;               /* [batch][n_head][head_dim], pool dtype */
  void* out;                   /* [batch][n_head * head_dim], out_dtype */
  int out_dtype;
  const int32_t* block_tables; /* [batch][max_blocks_per_seq] */
  int max_blocks_per_seq;
  const int32_t* context_lens; /* [batch], new token included */
  int max_context_len;
  int batch;
  const void* k_new;           /* new token's K/V stored by the call, or both NULL */
  const void* v_new;
} pkv_decode_batch;

int pkv_mixed_attention(pkv_pool* pool, int layer, const pkv_prefill_batch* prefill,
                        const pkv_decode_batch* decode, int n_head, float scale,
                        void* stream);
size_t pkv_mixed_workspace_bytes(const pkv_pool* pool, int n_head,
                                 const pkv_prefill_batch* prefill,
                                 const pkv_decode_batch* decode);

/* ---- rotary position embedding (crates/ai-engine-candle/src/paged/rope.rs,
 * applied per row in the decode step, transformer.rs:252-269) ---------------
 * Tables as Rope::new (rope.rs:14-23): theta_i = 1 / freq_base^(2 i / rope_dim)
 * in f32, angle[p][i] = (float)p * theta_i, cos/sin in f32, shape
 * [max_seq][rope_dim / 2].  The rotation is candle's rotate-half rope that
 * apply_rope uses (rope.rs:38-42): for the halves x1 = x[i], x2 = x[i + d/2]
 * of a head row, out[i] = x1 cos - x2 sin, out[i + d/2] = x1 sin + x2 cos,
 * in f32 with every product rounded (no fused multiply-add), then rounded to
 * the output dtype.  rope_dim is the head_dim of the rows it rotates. */
typedef struct pkv_rope pkv_rope;

/* Fills host arrays cos_host, sin_host [max_seq][rope_dim / 2] (host only). */
int pkv_rope_tables_host(int rope_dim, float freq_base, int max_seq,
                         float* cos_host, float* sin_host);
/* Tables computed on the host (as above) and kept in device memory. */
int pkv_rope_create(pkv_rope** out, int rope_dim, float freq_base, int max_seq,
                    int device);
int pkv_rope_destroy(pkv_rope* rope);
/* Device pointers of the tables (e.g. to share them with other kernels). */
int pkv_rope_tables(const pkv_rope* rope, const float** cos_dev,
                    const float** sin_dev);
/* x: [n_tokens][n_head][rope_dim] in in_dtype; out: same shape in out_dtype
 * (each PKV_F32, PKV_F16 or PKV_BF16; out may alias x when the dtypes
 * match).  positions: device int32 [n_tokens], token t rotated by row
 * positions[t] (Rope::gather, rope.rs:28-32).  A position outside
 * [0, max_seq) leaves that token's rows unwritten and makes the next
 * pkv_rope_check() report PKV_ERR_DEVICE_DATA. */
int pkv_rope_apply(pkv_rope* rope, const void* x, int in_dtype, void* out,
                   int out_dtype, const int32_t* positions, int n_tokens,
                   int n_head, void* stream);
int pkv_rope_check(pkv_rope* rope);

/* Decode attention with the rotary embedding applied inside the kernel: the
 * decode step's per-row RoPE of q and of the new k (transformer.rs:252-269)
 * followed by pkv_decode_attention (same arguments and results).  q and
 * k_new are the projections before rotation and v_new the new values, all
 * in in_dtype (PKV_F32 -- the reference's activations -- or the pool dtype);
 * the rotated q and k are rounded to the pool dtype, as stored k rows are.
 * positions: device int32 [batch] or NULL; NULL uses context_lens[b] - 1,
 * the reference's decode position (positions == seq_lens, engine.rs:130-133).
 * Given, they also bound the keys attended as in
 * pkv_decode_attention_positions (the reference's decode step passes the
 * same positions to the rotation and to build_mask, transformer.rs:237,290).
 * rope->rope_dim must equal the pool's head_dim.  A position outside
 * [0, max_seq) is reported by pkv_pool_check() and rotates by position 0. */
int pkv_decode_attention_rope(pkv_pool* pool, int layer, const pkv_rope* rope,
                              const int32_t* positions, int in_dtype,
                              const void* q, void* out, int out_dtype,
                              const int32_t* block_tables,
                              int max_blocks_per_seq,
                              const int32_t* context_lens, int max_context_len,
                              int batch, int n_head, float scale,
                              const void* k_new, const void* v_new,
                              void* stream);

/* The prefill step's glue in one launch (prefill_seq, transformer.rs:
 * 160-174: apply_rope to q and k, then KvPool::write of every token's k and
 * v, attention.rs:57-83): k rows rotated by positions[t] and v rows stored
 * at slot_mapping[t], as pkv_append; with q (not NULL), its rows rotated
 * into q_out for pkv_prefill_attention.
 *  k, v: [n_tokens][n_kv_head][head_dim], q: [n_tokens][n_head][head_dim],
 *  all in in_dtype (PKV_F32, PKV_F16 or PKV_BF16), 16-byte aligned; the
 *  stored rows and q_out are in the pool dtype (q_out may alias q when
 *  in_dtype is the pool dtype).  positions, slot_mapping: device int32
 *  [n_tokens]; slot < 0 skips that token's k/v (its q is still rotated).
 *  Rotation and rounding as pkv_rope_apply.  A position outside
 *  [0, max_seq) leaves that token's rotated rows unwritten and a slot
 *  beyond the pool its k/v; pkv_pool_check() reports either. */
int pkv_append_rope(pkv_pool* pool, int layer, const pkv_rope* rope,
                    const int32_t* positions, int in_dtype, const void* k,
                    const void* v, const int32_t* slot_mapping, int n_tokens,
                    const void* q, void* q_out, int n_head, void* stream);

/* ---- token selection (crates/ai-engine-runtime/src/sample.rs:12-55) --------
 * The engine copies each logits row to the host and samples it with
 * SamplingConfig {temperature of the request, top_p: None, top_k: None,
 * seed: 42} (crates/ai-engine-candle/src/paged/engine.rs:58-60,145-162,226);
 * this selects on the device and leaves one int32 per row.
 *  logits: device, row b at logits + b * row_stride elements, `vocab` values
 *  each, dtype PKV_F32 / PKV_F16 / PKV_BF16.  temperatures: device f32
 *  [batch], or NULL (every row greedy).  tokens: device int32 [batch].
 * Row b is argmax (first maximum; NaN never chosen; 0 when no value exceeds
 * -inf) when temperatures[b] == 0 or vocab <= 1.  Otherwise sample(): y =
 * logit / temperature sorted descending (ties in index order), the first
 * top_k kept (top_k == 0: None), p = softmax over them, the shortest prefix
 * whose cumulative p reaches top_p kept and renormalised (top_p >= 1 or NaN:
 * None), and the first token at which the cumulative p reaches r =
 * StdRng::seed_from_u64(seed).gen::<f32>() -- the same r on every call, as
 * in the reference.  The token equals the reference's except where its f32
 * running sums fall within their rounding of r or top_p.  Temperatures must
 * be finite and logits of sampled rows free of NaN (the reference's sort is
 * unspecified there).  vocab < 2^24 (probability masses are 2^-40 fixed
 * point summed in 64 bits).  Runs on the calling thread's current device.
 * Batches of at most 128 rows with temperatures and no top_k / top_p split
 * each row over G = min(32, 256 / batch, ceil(vocab / 4096)) workgroups,
 * with 57,624 + 4,096 G bytes per row of partial histograms (at most 184 KiB
 * per row; 1.5 MB for 8 rows, 8.4 MB for 128) in a stream-ordered allocation
 * on `stream` (capturable in a HIP graph); if that allocation fails, one
 * workgroup per row.  Both give the same tokens.  Scratch of this call and of
 * pkv_sample_exact comes from a memory pool of the library, which keeps up to
 * 512 MiB per device for the next call until pkv_sample_trim. */
int pkv_sample(const void* logits, int dtype, long long row_stride, int batch,
               int vocab, const float* temperatures, int top_k, float top_p,
               uint64_t seed, int32_t* tokens, void* stream);
/* sample() of crates/ai-engine-runtime/src/sample.rs:12-48 with the
 * reference's own f32 arithmetic, bit for bit: the token equals the
 * reference's on every row, including rows where its f32 rounding alone
 * moves the pick (pkv_sample matches those only to within that rounding).
 * Same arguments as pkv_sample except top_p: NaN is None and any other value
 * is Some(top_p), as in the reference, where Some(1.0) still truncates once
 * the f32 running sum reaches 1.  Exponentials are glibc's expf (what
 * f32::exp calls on x86-64 Linux), restated on the device and equal to the
 * host libm on every argument the path uses (<= 0); the order is, for f32
 * logits, buckets of y sorted only where a running sum needs the order
 * (rows that need more: a stable radix sort of every key), and for 16-bit
 * logits runs of equal values from a histogram of their 65,536 possible
 * keys; every f32 running sum (the softmax denominator, top_p's cumulative
 * sum, the r threshold) takes exactly the reference's rounding steps.
 * Scratch: 1 MB per row for f16/bf16 logits, 8 bytes per logit per row for
 * f32, at most 512 MB per launch (larger batches run in several launches),
 * in a stream-ordered allocation on `stream` (kept as pkv_sample's is, at most
 * 512 MiB in all until pkv_sample_trim).  One 1024-thread workgroup per
 * row; at most 64 rows of at least 65,536 f32 logits take min(32, 256 /
 * batch, ceil(vocab / 4096)) workgroups per row for the passes over the
 * logits (five launches, 0.2 MB more scratch per row, the same tokens). */
int pkv_sample_exact(const void* logits, int dtype, long long row_stride, int batch,
                     int vocab, const float* temperatures, int top_k, float top_p,
                     uint64_t seed, int32_t* tokens, void* stream);
/* pkv_sample_exact that also reports, for verification (no reference
 * counterpart), which kernel selected each row: routes (device int32
 * [batch]) gets 0 (argmax: temperature 0 or vocab <= 1), 1 (f32 logits:
 * buckets of y, sorted only where a running sum needs the order), 2 (runs
 * of equal 16-bit values; f32 rows whose logits are all bf16 values when
 * the buckets left them) or 3 (the radix sort of every logit).  Tokens are
 * those of pkv_sample_exact. */
int pkv_sample_exact_routes(const void* logits, int dtype, long long row_stride, int batch,
                            int vocab, const float* temperatures, int top_k, float top_p,
                            uint64_t seed, int32_t* tokens, int32_t* routes, void* stream);
/* The exp pkv_sample_exact uses, exposed for verification (no reference
 * counterpart): out[i] = expf(in[i]) as glibc computes it; device arrays of
 * n floats, on `stream`. */
int pkv_sample_expf(const float* in, float* out, long long n, void* stream);
/* Gives back the free scratch that pkv_sample and pkv_sample_exact keep on the
 * calling thread's current device (waits for the device; the next call
 * allocates again).  Every device allocation of this library does the same
 * when memory runs out (without the wait while its stream is captured). */
int pkv_sample_trim(void);
/* StdRng::seed_from_u64(seed).gen::<f32>() (sample.rs:41-42; host only). */
float pkv_sample_draw(uint64_t seed);

/* ---- speculative decoding over long contexts (no reference counterpart) ------
 * A step that drafts several tokens per request and attends to a chosen part
 * of each context, with lengths that stay on the device between steps:
 *   pkv_step_tables       block tables, slots and positions of the step
 *   pkv_append            its keys and values
 *   pkv_key_bounds        the bounds of the blocks that they filled
 *   pkv_select_blocks     per row and kv head, the blocks to attend
 *   pkv_sparse_attention  attention over them
 *   pkv_verify_drafts     the drafts that are kept and the token after them
 * All are stream-ordered, allocate nothing and can be captured in a HIP graph.
 * Scratch is the caller's (`workspace`, 16-byte aligned, of at least the bytes
 * that the query beside each call returns), so calls on several streams, or
 * several graphs, do not share any unless the caller makes them. */

/* Block tables, slots and positions of a step from lengths on the device: the
 * work of BlockAllocator::ensure_capacity and locate (block_table.rs:32-58) for a
 * whole step.  Request i has seq_lens[i] tokens in n_blocks[i] blocks
 * (block_tables[i][0 ..]; it may hold more blocks than it has tokens for) and
 * writes new_lens[i] more; blocks that it lacks are taken from the end of
 * free_list[0 .. *free_count - 1] in request order, as ensure_capacity does
 * request by request.
 *  block_tables, block_tables_out: int32 [n_seqs][max_blocks_per_seq] (entries past
 *      a request's blocks are written as 0); may be the same array.
 *  n_blocks_out: int32 [n_seqs], free_count_out: int32 [1], for the next step.
 *  context_lens: int32 [n_seqs] = seq_lens + new_lens; cu_q_lens: int32 [n_seqs + 1].
 *  positions, slot_mapping: int32 [max_tokens], token cu_q_lens[i] + t of request
 *      i at position seq_lens[i] + t; -1 past the step's tokens.  The slot of a
 *      block id outside [0, num_blocks) is INT32_MAX, which pkv_append reports.
 *  status: int32 [1].  0: done.  k > 0: the free list is k blocks short.  -1: a
 *      length is negative, a table too narrow, n_blocks or *free_count out of
 *      range (0 .. free_len), or the step has more than max_tokens tokens.
 *      Unless it is 0 nothing is allocated: tables, n_blocks and free_count
 *      are copied, context_lens = seq_lens, cu_q_lens 0, slots and positions -1.
 * Other outputs must not overlap the inputs or each other
 * (PKV_ERR_INVALID).  block_size: a power of two in [1, 256]; num_blocks *
 * block_size and max_blocks_per_seq * block_size below 2^31.  Runs on the calling
 * thread's current device. */
int pkv_step_tables(int block_size, int num_blocks, const int32_t* seq_lens,
                    const int32_t* new_lens, int n_seqs, const int32_t* block_tables,
                    const int32_t* n_blocks, int max_blocks_per_seq, const int32_t* free_list,
                    int free_len, const int32_t* free_count, int max_tokens,
                    int32_t* block_tables_out, int32_t* n_blocks_out, int32_t* free_count_out,
                    int32_t* context_lens, int32_t* cu_q_lens, int32_t* positions,
                    int32_t* slot_mapping, int32_t* status, void* stream);

/* Key bounds: [num_blocks][n_kv_head][2][head_dim] in the pool dtype, the
 * elementwise smallest, then largest, key element of each block and kv head (NaN
 * elements are passed over; +inf, then -inf, where all are NaN).  One array per
 * layer, of pkv_key_bounds_bytes, 16-byte aligned.  pkv_key_bounds brings those
 * of every block that holds a position from first_positions[s] (NULL: 0) to
 * context_lens[s] - 1 of a sequence up to date, from all of the block's keys below
 * context_lens[s].  max_new_len: host bound of context_lens[s] -
 * first_positions[s], 1 .. 2^30.  A sequence with lengths outside 0 <= first <=
 * context <= the table, or beyond max_new_len, is left out, as is a block id
 * outside the pool; pkv_pool_check() reports both.
 * A block that several sequences of a call share must have as many keys in
 * each. */
size_t pkv_key_bounds_bytes(const pkv_pool* pool);
int pkv_key_bounds(pkv_pool* pool, int layer, void* bounds, const int32_t* block_tables,
                   int max_blocks_per_seq, const int32_t* first_positions,
                   const int32_t* context_lens, int n_seqs, int max_new_len, void* stream);

/* The blocks that each query row attends, per kv head: the first first_blocks
 * and the last last_blocks of its context and, of those between, the ones with
 * the largest
 *     max over the group's heads h of  sum_d max(q_hd lo_d, q_hd hi_d),
 * an upper bound of q_h . k over the block's keys, top_blocks in all.  Exact: the
 * sums are compared as 64-bit ones, the lower index wins among equals.  A
 * context of at most top_blocks blocks is taken whole.
 *  q: [total_q][n_head][head_dim], pool dtype, as the attention will get it.
 *  cu_q_lens: int32 [n_seqs + 1], or NULL for one row per sequence (total_q ==
 *      n_seqs); context_lens: int32 [n_seqs].  As in pkv_prefill_attention row i of
 *      sequence s is at position context_lens[s] - q_len_s + i and has the keys
 *      up to that position; a row without keys gets no block.
 *  blocks: int32 [total_q][n_kv_head][top_blocks], indexes into the sequence's
 *      row of block_tables, ascending, then -1.  Rows of no sequence are left
 *      as they were.
 *  max_q_len, max_context_len: host upper bounds, 1 .. 2^30 (longer rows are
 *      left out, longer contexts cut off; pkv_pool_check() reports both).
 *  first_blocks >= 0, last_blocks >= 1, first_blocks + last_blocks <= top_blocks.
 * Only the bounds of blocks between the first and last ones are used, which are
 * full: the block that a step writes to needs none.  A block whose bounds are
 * not finite, one whose products' magnitudes add up past the f32 range, and any
 * block for a query that is not finite rank first (a NaN key that the bounds
 * passed over does not show).  Scores that differ by less than about
 * head_dim * 2^-126 may be ranked either way.  Block ids outside the pool are
 * reported by pkv_pool_check().  Workspace: about 12 bytes per row, kv head and
 * block of max_context_len. */
size_t pkv_select_workspace_bytes(const pkv_pool* pool, int n_seqs, int total_q, int max_q_len,
                                  int max_context_len, int max_blocks_per_seq, int n_head);
int pkv_select_blocks(pkv_pool* pool, const void* q, const void* bounds, int32_t* blocks,
                      int top_blocks, int first_blocks, int last_blocks,
                      const int32_t* cu_q_lens, const int32_t* context_lens,
                      const int32_t* block_tables, int max_blocks_per_seq, int n_seqs,
                      int total_q, int max_q_len, int max_context_len, int n_head,
                      void* workspace, size_t workspace_bytes, void* stream);

/* Attention of each query row over the keys of its listed blocks:
 * out_h = sum_k softmax_k(scale q_h . k) v_k, k over the keys of the row's context
 * that lie in blocks[row][kv head of h], f32 accumulation and softmax.  With every
 * block listed it is pkv_decode_attention (NULL cu_q_lens) or
 * pkv_prefill_attention, to rounding.
 *  q, out, out_dtype, scale (not NaN): as pkv_decode_attention; rows, cu_q_lens,
 *      context_lens, block_tables and max_q_len as pkv_select_blocks (rows of no
 *      sequence and those beyond max_q_len are left as they were).
 *  blocks: int32 [total_q][n_kv_head][top_blocks], distinct indexes in any order;
 *      negative entries are skipped.  An index past the row's context or a
 *      block id outside the pool is skipped and reported by pkv_pool_check().
 *      A row and kv head without any key is zero.  Attended keys and values are
 *      to be finite: with others that row and kv head may come out as NaN.
 * The launch has n_seqs * max_q_len row places, so max_q_len should be tight:
 * these, n_kv_head and the larger of parts (1 to top_blocks * block_size / 64) and,
 * where parts are merged by a second kernel, query heads per kv head (16 at most)
 * multiply to less than 2^26 (else PKV_ERR_UNSUPPORTED). */
size_t pkv_sparse_workspace_bytes(const pkv_pool* pool, int total_q, int n_head, int top_blocks);
int pkv_sparse_attention(pkv_pool* pool, int layer, const void* q, void* out, int out_dtype,
                         const int32_t* blocks, int top_blocks, const int32_t* cu_q_lens,
                         const int32_t* context_lens, const int32_t* block_tables,
                         int max_blocks_per_seq, int n_seqs, int total_q, int max_q_len,
                         int n_head, float scale, void* workspace, size_t workspace_bytes,
                         void* stream);

/* Verification of drafted tokens against the target's probabilities, from
 * given random numbers.  Request b has n = cu_drafts[b + 1] - cu_drafts[b] drafts d_i
 * and n + 1 target rows, rows cu_drafts[b] + b + i of target_logits; its draft rows
 * are cu_drafts[b] + i of draft_logits.  With p_i = softmax(target row i / T) and
 * q_i = softmax(draft row i / T), T = temperatures[b]:
 *   draft i is kept while uniforms[cu_drafts[b] + i] * q_i(d_i) < p_i(d_i);
 *   at the first that is not, the next token comes from max(p_i - q_i, 0), after
 *   the last draft from p_n: the first token at which the running sum of these
 *   weights passes final_uniforms[b] times their total.
 * draft_logits NULL: q_i is 1 at d_i (drafts that were looked up or searched).
 * T not positive or not finite, or temperatures NULL: greedy; a draft is kept
 * while it is the target row's first maximum, and the next token is a row's first
 * maximum.  Decisions are those of 64-bit arithmetic in which probabilities below
 * about 2^-1000 are 0; in a draw those below 2^-400 count as 0, and where nothing
 * is left of max(p_i - q_i, 0) the token comes from p_i.  A distribution cut by
 * top-k or top-p is given by its log-probabilities with -inf elsewhere, at
 * temperature 1.
 *  logits: rows of `vocab` values at a stride of row_stride elements, each side
 *      PKV_F32, PKV_F16 or PKV_BF16.  -inf has probability 0, and so has NaN; +inf
 *      counts as the largest f32 value.  A target row with nothing above -inf
 *      keeps no draft and ends with token 0.
 *  draft_tokens: int32 [total_drafts]; one outside [0, vocab) is not kept.
 *  cu_drafts: int32 [batch + 1], from 0 to total_drafts (a host value), nondecreasing.
 *  uniforms: f32 [total_drafts], final_uniforms: f32 [batch], in [0, 1); not read for
 *      greedy requests, nor the draft rows.  temperatures: f32 [batch].
 *  out_tokens: int32 [total_drafts + batch], at cu_drafts[b] + b the request's kept
 *      drafts, its next token, then -1.  n_accepted: int32 [batch], kept drafts.
 * Outputs and workspace must not overlap the inputs or each other
 * (PKV_ERR_INVALID).  vocab 1 .. 2^24 - 1.  Runs on the calling thread's current
 * device. */
size_t pkv_verify_workspace_bytes(int batch, int total_drafts, int vocab, int has_draft_logits);
int pkv_verify_drafts(const void* target_logits, int target_dtype, long long target_row_stride,
                      const void* draft_logits, int draft_dtype, long long draft_row_stride,
                      const int32_t* draft_tokens, const int32_t* cu_drafts, int batch,
                      int total_drafts, int vocab, const float* uniforms,
                      const float* final_uniforms, const float* temperatures,
                      int32_t* out_tokens, int32_t* n_accepted, void* workspace,
                      size_t workspace_bytes, void* stream);

/* ---- a cache held in 4 bits (no reference counterpart) ------------------------
 * A pool of dtype PKV_Q4 holds a third of what a 16-bit pool does for the same
 * tokens.  A step of an engine over one:
 *   pkv_prompt_attention  whole prompts over their own rows, before they are rounded
 *   pkv_q4_append         keys and values into the pool
 *   pkv_q4_attention      single tokens and chunks over the pool
 *   pkv_adjust_logits     penalties, biases and masks before pkv_sample
 * All are stream-ordered, allocate nothing and can be captured in a HIP graph;
 * scratch is the caller's.  Pool calls that do not read or write elements take such
 * pools too: shapes, pkv_pool_read / write / read_blocks (bytes), pkv_copy_blocks,
 * pkv_compact, pkv_pool_check.  The others return PKV_ERR_UNSUPPORTED.
 *
 * What is held: 32 neighbouring channels of a token's row in one kv head are a
 * group.  With its elements x (NaN taken as 0, others limited to +-65024), m =
 * f16(min x) and s = f16((max x - m) / 15), the subtraction and the division in f32,
 * an element is held as c = (x - m) / s in 64 bits, rounded to nearest even and
 * limited to 0 .. 15, and stands for m + s c.  Where s is not positive c is 0; s is
 * negative, and held so, where m rounds above max x.
 *
 * Layout: block_size a power of two in [16, 256], bs; hd = head_dim, G = hd / 32
 * groups, T = hd / 16.  One layer's K (or V) is [num_blocks][n_kv_head][chunk],
 * a chunk being bs * hd * 5 / 8 bytes:
 *   K  codes  [bs][4][G] 32-bit words: word (token, i, g) has channels 32 g + 8 i
 *             + e, e = 0 .. 7, in bits 4 (e / 2 + 4 (e % 2)) on
 *   V  codes  [bs / 4][16][4][T / 2] bytes: (token / 4, i, token % 4) has channels i + 16 t,
 *             t = 0 .. T - 1, in bits 4 t on
 *   both then s and m, each [bs / 4][G][4] f16 (token / 4, group, token % 4)
 * so that a token's bytes are its own: rows are written without reading others. */

/* Stores rows of k and v (dtype PKV_F32, PKV_F16 or PKV_BF16) in 4 bits: token i, at k +
 * i * k_token_stride elements (v likewise), [n_kv_head][head_dim], goes to slot
 * slot_mapping[i].  Slots as in pkv_append: negative ones are skipped, ones beyond
 * the pool reported by pkv_pool_check(); distinct (two tokens for one slot race).
 * Token strides: at least n_kv_head * head_dim, at most 2^24, a multiple of 16
 * bytes.  k and v 16-byte aligned. */
int pkv_q4_append(pkv_pool* pool, int layer, const void* k, const void* v, int dtype,
                  long long k_token_stride, long long v_token_stride,
                  const int32_t* slot_mapping, int n_tokens, void* stream);

/* The values that slots stand for: out_k, out_v [n][n_kv_head][head_dim] in out_dtype
 * (PKV_F32, PKV_F16 or PKV_BF16), 16-byte aligned.  A negative slot gives a zero row, one
 * beyond the pool a zero row that pkv_pool_check() reports. */
int pkv_q4_gather(pkv_pool* pool, int layer, const int32_t* slot_mapping, int n, void* out_k,
                  void* out_v, int out_dtype, void* stream);

/* Attention over a 4-bit pool: out_h = sum_k softmax_k(scale q_h . k) v_k over the
 * values that the row's keys stand for, f32 accumulation and softmax.  f32 queries are
 * f32 throughout.  With 16-bit queries weights enter the second product in 22 bits;
 * for up to 1024 / head_dim columns (rows times heads of a kv head) a product of a query element
 * and a code c is kept to 2^-17 of the largest of eight such elements;
 * in calls with a chunk of more than 32 columns values, and for bf16 queries also keys and
 * weights, may be rounded to f16.
 *  q: token i at q + i * q_token_stride elements, [n_head][head_dim] in q_dtype
 *      (PKV_F32, PKV_F16 or PKV_BF16); 16-byte aligned, the stride at least n_head *
 *      head_dim, at most 2^24 and a multiple of 16 bytes.  Elements beyond 2^100 in magnitude, or
 *      not finite, make their row's results undefined.
 *  out: [total_q][n_head * head_dim] in out_dtype (PKV_F32 or q_dtype), 16-byte aligned.
 *  cu_q_lens: int32 [n_seqs + 1], or NULL for one row per sequence (total_q ==
 *      n_seqs, max_q_len == 1); context_lens: int32 [n_seqs], the new tokens
 *      among them (appended before).  Row i of sequence s is at position context_lens[s] -
 *      q_len_s + i and has the keys up to it; a row without keys is zero.
 *  block_tables: int32 [n_seqs][max_blocks_per_seq].
 *  max_q_len, max_context_len: host upper bounds, 1 .. 2^30.  A sequence with a
 *      longer chunk or context, a context longer than its table, a negative
 *      length, or rows outside [0, total_q) is left out: its rows are as they
 *      were, as are rows of no sequence, and pkv_pool_check() reports it.  Keys of
 *      block ids outside the pool are not attended, and reported.
 *      A launch of 2^32 work-items is refused (PKV_ERR_UNSUPPORTED): 256 for each part of
 *      the keys (256 keys or more), sequence, kv head and 128 columns of max_q_len (total_q at
 *      most) times n_head / n_kv_head; 16 columns for f32 queries.
 *  n_head / n_kv_head: any integer.  scale finite.
 * Workspace: 16-byte aligned, of at least pkv_q4_workspace_bytes (0: none needed). */
size_t pkv_q4_workspace_bytes(const pkv_pool* pool, int n_seqs, int total_q, int max_q_len,
                              int max_context_len, int n_head);
int pkv_q4_attention(pkv_pool* pool, int layer, const void* q, int q_dtype,
                     long long q_token_stride, void* out, int out_dtype,
                     const int32_t* cu_q_lens, const int32_t* context_lens,
                     const int32_t* block_tables, int max_blocks_per_seq, int n_seqs,
                     int total_q, int max_q_len, int max_context_len, int n_head, float scale,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Causal attention of whole prompts over their own rows, packed: token i of prompt s
 * is row cu_lens[s] + i and attends tokens 0 .. i of its prompt; out_h = sum_j
 * softmax_j(scale q_h . k_j) v_j, f32 accumulation and softmax (for 16-bit types the
 * weights are rounded to them before the second product).  Tokens behind i may hold
 * anything, NaN and infinities too.
 *  q: token t at q + t * q_token_stride elements, [n_head][head_dim]; k, v likewise,
 *      [n_kv_head][head_dim]; all in dtype (PKV_F32, PKV_F16 or PKV_BF16), 16-byte
 *      aligned, strides multiples of 16 bytes that hold a row, at most 2^24.  Query head h reads kv head
 *      h / (n_head / n_kv_head).  head_dim 64, 128 or 256.
 *  out: [total][n_head * head_dim] in out_dtype (PKV_F32 or dtype), 16-byte aligned; may not
 *      overlap q, k or v.
 *  cu_lens: int32 [n_seqs + 1], nondecreasing, within 0 .. total; a prompt that
 *      breaks this is left out.  Rows of no prompt are left as they were.
 *  max_len: host bound of the prompt lengths, 1 .. 2^30; longer prompts are computed too,
 *      with fewer workgroups than they could use.  scale finite.
 * Runs on the calling thread's current device. */
int pkv_prompt_attention(const void* q, const void* k, const void* v, int dtype,
                         long long q_token_stride, long long k_token_stride,
                         long long v_token_stride, void* out, int out_dtype,
                         const int32_t* cu_lens, int n_seqs, int total, int max_len, int n_head,
                         int n_kv_head, int head_dim, float scale, void* stream);

/* Logits before a token is chosen: with n = how often token t is among the generated
 * tokens of request b, in f32, each operation rounded, and once to dtype at the end:
 *   x = logits[b][t]
 *   t among the request's tokens:  x = x > 0 ? x / r : x * r    r = repetition[b]
 *   n > 0:                         x = x - frequency[b] * n; x = x - presence[b]
 *   t among its biased tokens:     x = x + its bias (the last entry of t counts)
 *   t without its mask bit:        x = -inf
 *  logits: [batch] rows of `vocab` values at row_stride elements, PKV_F32, PKV_F16 or
 *      PKV_BF16; out: the same type at out_row_stride; may be logits itself (with the
 *      same stride), may not overlap it otherwise.
 *  tokens: int32 [total_tokens], request b's at cu_tokens[b] .. cu_tokens[b + 1] - 1, the
 *      first prompt_lens[b] of them (NULL: none) its prompt; NULL (with cu_tokens): none.
 *  repetition, presence, frequency: f32 [batch] or NULL (1, 0, 0).  r not positive or
 *      not finite counts as 1.
 *  bias_tokens, bias_values: int32, f32 [total_bias], request b's at cu_bias[b] ..
 *      cu_bias[b + 1] - 1; all three NULL: none.
 *  mask: uint32 [n_masks][mask_row_words], bit t % 32 of word t / 32 set where t may be
 *      chosen; NULL: none.  mask_rows: int32 [batch], the row of a request, negative: no
 *      mask, n_masks or more: nothing may be chosen; NULL: row b.
 * Token ids outside [0, vocab) are passed over; offsets are limited to the arrays (at
 * most 2^30 entries) and a request whose offsets decrease has no entries.  vocab
 * 1 .. 2^24 - 1.
 * Runs on the calling thread's current device. */
int pkv_adjust_logits(const void* logits, void* out, int dtype, long long row_stride,
                      long long out_row_stride, int batch, int vocab, const int32_t* tokens,
                      const int32_t* cu_tokens, int total_tokens, const int32_t* prompt_lens,
                      const float* repetition, const float* presence, const float* frequency,
                      const int32_t* bias_tokens, const float* bias_values,
                      const int32_t* cu_bias, int total_bias, const uint32_t* mask, int n_masks,
                      int mask_row_words, const int32_t* mask_rows, void* stream);

/* Kernel timing (instrumentation; no reference counterpart).  While enabled,
 * every pkv_decode_attention, pkv_prefill_attention, pkv_copy_blocks and
 * pkv_compact call records HIP events, owned by the pool, on its stream right
 * before and right after its main kernel -- the partition kernel of decode,
 * not its split-context merge; the one kernel of the others (for compaction,
 * after the plan upload).  pkv_pool_profile_read synchronises,
 * returns the summed main-kernel time in ms and the number of timed
 * launches since the last read, and clears the record. */
int pkv_pool_profile(pkv_pool* pool, int enable);
int pkv_pool_profile_read(pkv_pool* pool, double* total_ms, int* launches);

/* Synchronise the pool's device and report (then clear) any out-of-range
 * slot/block id or length a kernel met since the last check:
 * PKV_OK or PKV_ERR_DEVICE_DATA. */
int pkv_pool_check(pkv_pool* pool);

/* ---- host block bookkeeping (BlockAllocator / BlockTable,
 * block_table.rs:5-58).  Pure host code, usable without a GPU. ------------ */
typedef struct pkv_allocator pkv_allocator;
typedef struct pkv_table pkv_table;

/* BlockAllocator::new: free list [num_blocks-1, ..., 1, 0], pops from the end
 * so the first blocks handed out are 0, 1, 2, ... (block_table.rs:17-21). */
pkv_allocator* pkv_allocator_new(size_t num_blocks, size_t block_size);
void pkv_allocator_free(pkv_allocator* a);
size_t pkv_allocator_free_count(const pkv_allocator* a);       /* :23-25 */
size_t pkv_allocator_blocks_for(const pkv_allocator* a, size_t n_tokens); /* :27-30 */
/* :32-47  PKV_OK, or PKV_ERR_CAPACITY with nothing allocated. */
int pkv_allocator_ensure_capacity(pkv_allocator* a, pkv_table* t,
                                  size_t n_tokens);
/* :49-52  appends the table's blocks to the free list in table order. */
void pkv_allocator_release(pkv_allocator* a, pkv_table* t);
/* :54-58  PKV_ERR_INVALID when pos is beyond the table (the reference panics). */
int pkv_allocator_locate(const pkv_allocator* a, const pkv_table* t,
                         size_t pos, uint32_t* block_id, size_t* slot);

pkv_table* pkv_table_new(void);
void pkv_table_free(pkv_table* t);
size_t pkv_table_len(const pkv_table* t);
const uint32_t* pkv_table_blocks(const pkv_table* t);

/* ---- continuous-batching scheduler (run_loop / prefill block bookkeeping,
 * crates/ai-engine-candle/src/paged/engine.rs:62-237).  Pure host code.
 *
 * The reference's engine thread interleaves scheduling with the model; here
 * the scheduling is a step machine the caller drives around its own model
 * forward:  pkv_sched_step() returns the plan of the next forward (rows, block
 * tables, context lengths, slot mappings, copy-on-write copies), the caller
 * runs the layers (pkv_copy_blocks, pkv_append / pkv_decode_attention /
 * pkv_prefill_attention), samples one token per producing row and hands them
 * to pkv_sched_complete().  What the reference sends on a request's channel
 * (Ok(token) / Err(message) / channel closed) comes back as events.
 *
 * prefill_chunk == 0 reproduces run_loop exactly: an iteration first admits
 * requests (engine.rs:77-100) and prefills each whole prompt (a plan of
 * prefill rows), then runs the capacity/eviction pass and one decode step for
 * every running sequence (engine.rs:102-178, a plan of decode rows).
 * prefill_chunk > 0 is chunked prefill: each step carries the next chunk of
 * every prompt in flight (at most step_token_budget prompt tokens) together
 * with the decode rows.  Extensions with no reference counterpart: fork
 * (shared blocks under reference counts; the first write to a shared block
 * copies it, reported in the plan) and compaction (live blocks renumbered to
 * [0, live) with the fewest moves, returned for pkv_compact). */
typedef struct pkv_sched pkv_sched;

typedef struct {
  int max_num_seqs;      /* EngineConfig (engine.rs:30-36) */
  int block_size;
  int kv_cache_blocks;
  int max_seq;
  int32_t eos_token_id;
  int prefill_chunk;     /* 0: whole prompts (the reference) */
  int step_token_budget; /* chunked mode: prompt tokens per step (0: none) */
} pkv_sched_config;

#define PKV_EV_TOKEN 0    /* Ok(token) */
#define PKV_EV_FINISHED 1 /* the sequence ended; its blocks are released */
#define PKV_EV_ERROR 2    /* Err(message); the sequence ended */

typedef struct {
  int64_t seq;
  int kind;
  int32_t token;
  char message[120];
} pkv_sched_event;

/* One forward's plan; the arrays stay valid until the next step, complete,
 * fork or compact call.  Rows are the prefill rows, then the decode rows. */
typedef struct {
  int n_prefill, n_decode, n_rows, max_blocks, n_tokens, n_copies;
  const int64_t* row_seq;       /* [n_rows] */
  const int32_t* block_tables;  /* [n_rows][max_blocks], 0-padded */
  const int32_t* context_lens;  /* [n_rows] keys attended after the writes */
  const int32_t* cu_q_lens;     /* [n_prefill + 1] offsets of prompt tokens */
  const int32_t* q_start;       /* [n_prefill] position of each chunk's first token */
  const int32_t* slot_mapping;  /* [n_tokens] chunk tokens, then one per decode row */
  const int32_t* positions;     /* [n_tokens] position of each new token */
  const int8_t* produces;       /* [n_rows] 1 if the row yields a token */
  const int32_t* copy_src;      /* [n_copies] copy before the writes */
  const int32_t* copy_dst;
} pkv_sched_plan;

/* Message of the calling thread's last failed pkv_sched_* call. */
const char* pkv_sched_last_error(void);
int pkv_sched_create(pkv_sched** out, const pkv_sched_config* cfg);
void pkv_sched_destroy(pkv_sched* s);
/* GenRequest (engine.rs:13-18) without the channel; *id names its events. */
int pkv_sched_submit(pkv_sched* s, int prompt_len, int max_tokens, int64_t* id);
/* Plans the next forward; n_rows == 0 means nothing is runnable. */
int pkv_sched_step(pkv_sched* s, pkv_sched_plan* plan);
/* tokens: one per producing row, in row order (n = their count).  error !=
 * NULL reports a failed forward: every row's sequence ends with Err (the
 * reference's "prefill: ..." / "forward: ..." paths). */
int pkv_sched_complete(pkv_sched* s, const int32_t* tokens, int n,
                       const char* error);
/* Next event; returns 1 and fills *ev, or 0 when there is none. */
int pkv_sched_poll(pkv_sched* s, pkv_sched_event* ev);
/* Fork a decoding sequence: the child shares its blocks (copy-on-write) and
 * continues from the same position and pending token. */
int pkv_sched_fork(pkv_sched* s, int64_t parent, int max_tokens, int64_t* child);
/* Renumber live blocks to [0, live); src/dst (capacity cap) receive the moves
 * for pkv_compact, *n their count. */
int pkv_sched_compact(pkv_sched* s, int32_t* src, int32_t* dst, int cap, int* n);
/* Introspection: counts, a sequence's table (NULL if it is not live). */
int pkv_sched_counts(const pkv_sched* s, int* running, int* waiting,
                     int* free_blocks);
int pkv_sched_table(const pkv_sched* s, int64_t seq, const uint32_t** blocks,
                    int* n_blocks, int* pos);

#ifdef __cplusplus
}
#endif

#endif /* PAGEDKV_H */
