/*
 * eesd.h — C ABI of the B200 (sm_100a) kernels for the packed, ragged LayerSkip-Llama
 * draft/verify step.
 *
 * Conventions
 *   - Every pointer argument is a DEVICE pointer unless marked "host".
 *   - `stream` is a cudaStream_t passed as void*.  Nothing here synchronises the stream,
 *     allocates device memory or frees it: the caller owns every buffer.
 *   - Every function returns an int status (EESD_OK = 0).  Argument errors are detected on
 *     the host before any launch; device-side faults of the data (an out-of-range row,
 *     position or token id) and bounded-wait timeouts are OR-ed into a device status word
 *     that eesd_model_check() / eesd_status_read() return.
 *   - Element types: EESD_BF16 or EESD_F32 (the model dtype; tcgen05 GEMMs serve bf16, a
 *     CUDA-core FFMA GEMM serves the fp32 parity path).
 *   - Token ids, positions and cache rows are int32.
 *
 * Packed batch (the reference's `PackedBatch`, solutions/packed.py:63-78): tokens of
 * several request blocks are concatenated on one axis; block b holds T_b consecutive
 * tokens at positions pos0_b .. pos0_b+T_b-1 of KV-cache row row_b.  A query at position
 * p of row r attends to cached positions <= p of row r after this call's K/V are written
 * (solutions/packed.py:6-8).
 */
#ifndef EESD_H
#define EESD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define EESD_OK 0
#define EESD_ERR_ARG 1         /* invalid argument or unsupported shape (nothing launched)  */
#define EESD_ERR_CUDA 2        /* a CUDA runtime / driver call failed                       */
#define EESD_ERR_DEVICE 3      /* the device status word is non-zero (see eesd_status_*)    */

#define EESD_BF16 0
#define EESD_F32 1

/* GEMM epilogues (y[t, o] for token t, output feature o) */
#define EESD_EPI_STORE 0       /* y = acc                                                   */
#define EESD_EPI_RESIDUAL 1    /* y = residual + round(acc)   (x + F.linear(...))           */
#define EESD_EPI_SWIGLU 2      /* y = silu(round(g)) * round(u), g/u = rows o and o+up_offset */

/* Launch categories for the optional per-kernel CUDA-event profile */
#define EESD_PROF_NORM 0
#define EESD_PROF_GEMM_QKV 1
#define EESD_PROF_ROPE_KV 2
#define EESD_PROF_ATTN 3
#define EESD_PROF_GEMM_O 4
#define EESD_PROF_GEMM_W13 5
#define EESD_PROF_GEMM_W2 6
#define EESD_PROF_HEAD 7
#define EESD_PROF_MISC 8
#define EESD_PROF_KINDS 9

/* Library version and the text of the last host-side error of the calling thread. */
int eesd_version(void);
const char* eesd_last_error(void);

/* ------------------------------------------------------------------------------------ */
/* Model runtime.  Replaces the weight/KV layout of LayerSkipLlama (common/model.py:161-183,
 * 222-293) and the per-layer loop of packed_layers (solutions/packed.py:169-196).        */

typedef struct EesdModelDesc {
  int32_t dtype;                 /* EESD_BF16 | EESD_F32 */
  int32_t n_layers, dim, n_heads, n_kv_heads, head_dim, intermediate, vocab;
  float norm_eps;
  int32_t max_batch;             /* KV-cache rows */
  int32_t max_seq;               /* positions per row (multiple of 64) */
  int32_t max_tokens;            /* largest packed token count of one call */
  int32_t weights_packed;        /* bf16 only: 1 = wqkv, wo, w13, w2 and lm_head point to tile-packed
                                    copies (eesd_pack_weight), read as contiguous 16 KB tiles */
  /* per-layer weights: arrays (host memory) of n_layers device pointers */
  const void* const* wqkv;       /* [(Hq + 2 Hkv) D, dim] rows = [q; k; v] (common/model.py:262-263) */
  const void* const* wo;         /* [dim, Hq D] */
  const void* const* w13;        /* [2 I, dim] rows = [gate; up] (common/model.py:264-265) */
  const void* const* w2;         /* [dim, I] */
  const void* const* attn_norm;  /* [dim] */
  const void* const* ffn_norm;   /* [dim] */
  const void* final_norm;        /* [dim] */
  const void* lm_head;           /* [vocab, dim] (the embedding when tied) */
  const void* embed;             /* [vocab, dim] */
  const float* rope_cos;         /* [max_seq, D] fp32, rotate-half layout (common/model.py:129-140) */
  const float* rope_sin;
  void* k_cache;                 /* [n_layers, max_batch, Hkv, max_seq, D] (common/model.py:171-179) */
  void* v_cache;
  void* workspace;               /* eesd_model_workspace_bytes() bytes, 256-byte aligned */
  size_t workspace_bytes;
} EesdModelDesc;

/* One packed call (PackedBatch, solutions/packed.py:63-139, minus buckets and masks). */
typedef struct EesdBatch {
  int32_t n_tokens;
  int32_t n_blocks;
  int32_t n_items;               /* attention work items (block, query tile) */
  int32_t max_ctx;               /* host: max over blocks of pos0 + T */
  const int32_t* tok_pos;        /* [n_tokens] absolute position of every token */
  const int32_t* tok_row;        /* [n_tokens] KV-cache row of every token */
  const int32_t* blk;            /* [n_blocks, 4] = (start, T, row, pos0) */
  const int32_t* items;          /* [n_items, 2] = (block, first token within block) */
} EesdBatch;

/* Tile-packed weight layout for the bf16 GEMMs: a [rows, k] row-major bf16 matrix (k % 64 == 0)
 * becomes [ceil(rows/128) * k/64][128][64]: the 128 x 64 operand tile (row tile m, k-block j) is
 * the contiguous 16 KB block m * (k/64) + j, so each CTA streams its weights sequentially from HBM
 * (rows past the end are zero).  Layout change only; the GEMM numerics are unchanged.  w13 needs
 * intermediate % 128 == 0 to be packed as one matrix. */
size_t eesd_packed_weight_bytes(int rows, int k);
int eesd_pack_weight(const void* w, int rows, int k, void* out, void* stream);

/* Query tokens per attention work item for a model (items tile every block by this). */
int eesd_attn_item_tokens(int n_heads, int n_kv_heads);

size_t eesd_model_workspace_bytes(const EesdModelDesc* desc);
int eesd_model_create(const EesdModelDesc* desc, void** handle_out);
int eesd_model_destroy(void* handle);

/* Layers [start, end) on the packed hidden states x [n_tokens, dim] (in place), writing this
 * call's K/V into the cache.  solutions/packed.py:169-196 (packed_layer / packed_layers). */
int eesd_forward_layers(void* handle, void* x, const EesdBatch* batch, int start, int end, void* stream);

/* Shared exit head: final RMSNorm + LM head + greedy argmax over rows `rows` (nullable =
 * 0..n-1) of x.  common/model.py:328-330 with solutions/engine.py:352,463 (argmax).
 * out_ids [n] int32; logits (nullable) [n, vocab] in the model dtype. */
int eesd_head_argmax(void* handle, const void* x, const int32_t* rows, int n, int32_t* out_ids, void* logits,
                     void* stream);

/* x[i] = embed[ids[i]] (common/model.py:325-326), ids [n] int32. */
int eesd_embed(void* handle, const int32_t* ids, int n, void* x, void* stream);

/* Copy the device status word of the model to the host (synchronous on `stream`) and clear
 * it.  Returns EESD_ERR_DEVICE when any bit was set; *bits_out (host, nullable) gets them. */
int eesd_model_check(void* handle, int* bits_out, void* stream);

/* Per-kernel CUDA-event timing of the runtime's launches (off by default).  enable=1 starts a
 * new window; read fills ms[EESD_PROF_KINDS] and launches[EESD_PROF_KINDS] (host arrays) after
 * synchronising the recorded events. */
int eesd_model_profile(void* handle, int enable);
int eesd_model_profile_read(void* handle, double* ms, int64_t* launches);

/* The recorded launches one by one (kind, packed token count, ms), at most `cap` (host
 * arrays, each nullable); returns the number written, or -1 on error. */
int eesd_model_profile_records(void* handle, int32_t* kinds, int32_t* n_tok, float* ms, int cap);

/* Number of kernel launches the runtime issued since creation (host counter). */
int64_t eesd_model_launch_count(void* handle);

/* ------------------------------------------------------------------------------------ */
/* Step kernels of the EESD engine.  solutions/engine.py:345-352, 453-475.              */

/* dst[i, :] = src[src_idx[i], :] (src_idx nullable = i); dst_idx (nullable = i) scatters. */
int eesd_copy_rows(int dtype, const void* src, const int32_t* src_idx, void* dst, const int32_t* dst_idx, int n,
                   int width, void* stream);

/* ids[i] = table[idx[i]] (int32 gather, e.g. input ids from the token buffer seq_buf). */
int eesd_gather_ids(const int32_t* table, const int32_t* idx, int32_t* ids, int n, void* stream);

/* ids scatter: table[idx[i]] = ids[i] (e.g. drafts into seq_buf). */
int eesd_scatter_ids(const int32_t* ids, const int32_t* idx, int32_t* table, int n, void* stream);

/* Greedy acceptance (solutions/engine.py:464-475; common/engine.py:386-388).  For verifier v
 * with vinfo[v] = (start, T, slot): the verified tokens are y[start .. start+T-1] and the
 * drafts are seq_buf[slot * stride + 1 .. T-1].  acc[v] = first j < T-1 with
 * y[start+j] != draft j (else T-1); seq_buf[slot * stride] = y[start + acc[v]]. */
int eesd_greedy_accept(const int32_t* y, const int32_t* vinfo, int nv, int32_t* seq_buf, int stride, int32_t* acc,
                       void* stream);

/* Device-built metadata of one synchronous draft/verify round (gamma drafts + 1 verify), so the
 * host can enqueue round r+1 before it reads round r's acceptance (the reference's host packing,
 * solutions/packed.py:81-139, and position update, solutions/engine.py:373-396, done on the GPU).
 * act [n]: the round's cache rows; pos [max_batch]: round-start position per row.  out holds
 * eesd_round_meta_ints(n, gamma, item_tokens) int32, cols = gamma + 1, ni = ceil(cols/item_tokens):
 *   shallow step j = 0..cols-1 at j * 10 n: tok_pos [n] = pos + j, tok_row [n], blk [n, 4] =
 *     (i, 1, row, pos + j), items [n, 2] = (i, 0), src [n] = row * cols + j, dst [n] = src + 1
 *   verify at cols * 10 n: tok_pos [n cols], tok_row [n cols], blk [n, 4] = (i cols, cols, row,
 *     pos), items [n ni, 2], rows [n cols] = row * cols + t, vinfo [n, 3] = (i cols, cols, row)
 * eesd_round_advance: pos[act[i]] += acc[i] + 1 (rollback by length, solutions/engine.py:12-14). */
size_t eesd_round_meta_ints(int n, int gamma, int item_tokens);
int eesd_round_meta(const int32_t* act, int n, const int32_t* pos, int max_batch, int gamma, int item_tokens,
                    int32_t* out, void* stream);
int eesd_round_advance(const int32_t* act, int n, const int32_t* acc, int32_t* pos, int max_batch, void* stream);

/* ------------------------------------------------------------------------------------ */
/* Primitive kernels (exported for tests and for callers composing their own step).    */

/* y[i] = rms_norm(x[rows ? rows[i] : i]) * w   (common/model.py:153-156) */
int eesd_rmsnorm(int dtype, const void* x, const int32_t* rows, const void* w, void* y, int n, int dim, float eps,
                 void* stream);

/* Varlen GQA attention of one packed batch over ONE layer's KV cache.  solutions/packed.py:142-166
 * (`_attend`: per-bucket SDPA over [b, Hkv, G T, D] queries with a bool mask) without buckets or
 * masks: query (token t of block b, head h) attends to positions <= pos0_b + t of row row_b.
 * qkv [n_tokens, (Hq + 2 Hkv) D] is the fused projection output (q heads first, then k, then v);
 * k_cache / v_cache [max_batch, Hkv, max_seq, D]; out [n_tokens, Hq D].  The batch's `items` tile
 * every block into work items of eesd_attn_item_tokens() tokens (tok_pos / tok_row are unused).
 * append = 0: q is used as given (already rotated) and the cache already holds this call's keys.
 * append = 1 (bf16, every block one item, no two blocks on the same cache row): the kernel applies
 * RoPE (rope_cos / rope_sin [max_seq, D] fp32, solutions/packed.py:176-177) to q and k and writes k,
 * v at (row, position) first (solutions/packed.py:180-181).  Each work item appends only its own
 * block's keys, so a row's blocks must come in separate calls (or use eesd_rope_kv_append first).  An item whose block lies outside the batch or whose positions lie
 * outside its row sets a bit in *status (device int32, nullable) and is skipped. */
int eesd_attn_varlen_gqa(int dtype, const void* qkv, int n_heads, int n_kv_heads, int head_dim, void* k_cache,
                         void* v_cache, int max_batch, int max_seq, const EesdBatch* batch, int append,
                         const float* rope_cos, const float* rope_sin, void* out, int32_t* status, void* stream);

/* RoPE of q and k and the in-place KV append of a packed batch (common/model.py:143-150 apply_rope,
 * solutions/packed.py:176-181): q rotated in place in qkv, rotated k and v written to
 * k_cache / v_cache [max_batch, Hkv, max_seq, D] at (tok_row[t], tok_pos[t]).  A token whose row or
 * position is out of range sets a bit in *status (nullable) and is skipped. */
int eesd_rope_kv_append(int dtype, void* qkv, const int32_t* tok_pos, const int32_t* tok_row, int n_tok, int n_heads,
                        int n_kv_heads, int head_dim, const float* rope_cos, const float* rope_sin, void* k_cache,
                        void* v_cache, int max_batch, int max_seq, int32_t* status, void* stream);

/* y[n_tok, n_out] = epilogue(x[n_tok, k] @ w[n_out(+up), k]^T).  workspace: see
 * eesd_gemm_workspace_bytes (split-K partials and tile counters; zeroed by this call). */
size_t eesd_gemm_workspace_bytes(int n_tok, int n_out, int k, int epilogue);
int eesd_gemm(int dtype, int epilogue, const void* x, const void* w, const void* residual, void* y, int n_tok,
              int n_out, int k, int up_offset, void* workspace, size_t workspace_bytes, void* stream);

/* Tuning knobs.  EESD_OPT_MMA_N: N of one tcgen05.mma in the bf16 GEMM (0 = the whole token
 * tile, else a fixed multiple of 16 up to 256); numerics-neutral by design.  EESD_OPT_SPLITS:
 * split-K count (0 = derived from the weight shape; any fixed value keeps batch invariance but
 * changes the summation order, so AR and speculative runs must use the same value).
 * EESD_OPT_STAGES: TMA pipeline depth (0 = as many stages as fit; numerics-neutral).
 * EESD_OPT_PAIR: 1 (default) runs SwiGLU GEMMs on CTA pairs (cta_group::2, M = 256) where the
 * weight shape allows, 0 on single CTAs; AR and speculative runs must use the same value.
 * EESD_OPT_HEAD_TWO_TILES: 1 (default) lets an LM-head launch of up to 256 tokens take two
 * 128-row tiles per CTA (two accumulators), 0 one; numerics-neutral. */
#define EESD_OPT_MMA_N 1
#define EESD_OPT_SPLITS 2
#define EESD_OPT_STAGES 3
#define EESD_OPT_PAIR 4
#define EESD_OPT_HEAD_TWO_TILES 5
/* EESD_OPT_SPIN_LIMIT (tests of the failure path): poll limit of the pipeline waits of the GEMM and
 * attention kernels launched afterwards; -1 restores the default (2^24 polls), 0 makes every such
 * wait give up at once.  A wait that gives up sets a timeout bit in the device status word, the
 * kernel lets the copies and MMAs it already issued land, and returns. */
#define EESD_OPT_SPIN_LIMIT 6
/* EESD_OPT_MMA_SPLIT: a bf16 GEMM token tile above 256 tokens on one CTA takes two MMAs per K16
 * step; this sets the first one's N (a multiple of 16, default 192), the second takes the rest.
 * 0 = two equal halves.  Numerics-neutral. */
#define EESD_OPT_MMA_SPLIT 7
int eesd_set_option(int option, int value);

/* Exit head that allocates nothing, for callers that cannot call cudaMalloc (a serving
 * runtime whose allocator is locked on its decode path, code inside a foreign stream capture, a
 * plug-in that only receives input/output pointers).  No counterpart in the reference: it is the
 * same computation as eesd_head_argmax (final RMSNorm with norm_w, LM head, greedy argmax of rows
 * `rows` (nullable = 0..n-1) of x [x_rows, dim] bf16 -> out_ids [n] int32) without a model handle
 * or workspace.  Its scratch is a fixed 2 MiB + 1280 B __device__ array inside the library, held
 * by every GPU that loads the library until exit.  Limits: bf16, 1 <= n <= 128, dim a multiple of
 * 64 up to 8192; larger sizes return EESD_ERR_ARG with a message.  `stream` must belong to the
 * current device.  The first call on a device resolves the array's device address
 * (cudaGetSymbolAddress) and should come before any stream capture.  All calls share the array:
 * calls that overlap on the GPU race and must be serialised by the caller.
 * Device-side errors: a row index outside [0, x_rows) or a bounded wait that gave up makes every
 * out_id -1, and the call's status bits (0 = none) are written to *status_out (device int32,
 * nullable), both on the stream. */
int eesd_head_argmax_static(const void* x, int x_rows, const int32_t* rows, int n, int dim, int vocab,
                            const void* norm_w, const void* lm_head, float eps, int32_t* out_ids,
                            int32_t* status_out, void* stream);

/* ------------------------------------------------------------------------------------ */
/* Tree drafts and 8-bit KV caches: primitives for a draft/verify step whose drafts form a tree, over a
 * cache in the model dtype or in 8 bits.  The reference drafts chains over an unquantised cache
 * (solutions/packed.py:142-196, solutions/engine.py:453-475); with chains and EESD_KV_MODEL these calls
 * compute what eesd_rope_kv_append, eesd_attn_varlen_gqa and eesd_greedy_accept compute.
 *
 * One round: eesd_tree_meta once; per layer eesd_kv_append, then eesd_attn_tree; after the head
 * eesd_tree_accept, then eesd_kv_compact over all layers (the accepted path's K/V move to the front, so
 * that positions ctx .. ctx + n_acc of every row hold the path; rollback stays a length reset). */

#define EESD_KV_MODEL 0        /* elements of the model dtype (EESD_BF16 or EESD_F32) */
#define EESD_KV_E4M3 1         /* 8-bit floats (4 exponent, 3 mantissa bits), max 448; the NaN pattern is never stored */
#define EESD_KV_INT8 2         /* 8-bit integers -127 .. 127 */

/* 8-bit formats: K and V each have one power-of-two scale 2^e per (row, KV head, slot), stored as the
 * byte e + 127.  e is the smallest integer with max|x| <= Q 2^e (Q = 448 or 127) and e >= -100; the
 * stored element is x 2^-e rounded to nearest even, so every element is within half a step of x and
 * reads back exactly into bf16.  A vector with an infinity or NaN stores byte 255 and zeros, and reads
 * back as NaN. */
typedef struct EesdKvCache {
  int32_t format;                /* EESD_KV_* */
  int32_t n_layers, max_batch, n_kv_heads, max_seq, head_dim;   /* head_dim 64 or 128 */
  void* k;                       /* [n_layers, max_batch, Hkv, max_seq, D], 16-byte aligned */
  void* v;
  uint8_t* k_exp;                /* [n_layers, max_batch, Hkv, max_seq], 16-byte aligned; 8-bit formats only */
  uint8_t* v_exp;
} EesdKvCache;

#define EESD_TREE_MAX_NODES 256  /* nodes per block with a visibility mask (or eesd_tree_accept) */

/* Blocks of tree nodes.  Block b: T nodes of cache row `row` behind `ctx` committed positions; node i
 * sits at cache slot ctx + i.  A tree's nodes are numbered so that parent[i] < i (indices within the
 * block; -1 for a node whose parent is the committed context). */
typedef struct EesdTree {
  int32_t n_tokens, n_blocks;
  int32_t max_nodes;             /* host: largest T, at least */
  int32_t max_ctx;               /* host: largest ctx + T, at least (<= max_seq) */
  int32_t words;                 /* 64-bit words per mask row: (max_nodes + 63) / 64, at most 4; 0 without a mask */
  int32_t reserved;              /* 0 */
  const int32_t* blk;            /* [n_blocks, 4] = (start, T, row, ctx), 16-byte aligned; no two blocks
                                    share a token, tokens of no block are padding */
  const int32_t* parent;         /* [n_tokens], NULL: every block is a chain */
  int32_t* tok_pos;              /* [n_tokens] RoPE position: ctx + depth */
  int32_t* tok_slot;             /* [n_tokens] cache slot: ctx + i */
  int32_t* tok_row;              /* [n_tokens] cache row */
  uint64_t* mask;                /* [n_tokens, words]: bit j of node i's row: i sees node j of its block.  NULL:
                                    causal, i sees nodes 0 .. i.  Any mask works in eesd_attn_tree. */
} EesdTree;

/* tok_pos, tok_slot, tok_row and (unless NULL) mask from blk and parent, on the device: a node sees its
 * ancestors and itself.  A block outside the tokens or the cache, or a parent that does not come before
 * its node, sets a bit in *status (device int32, nullable); the tokens of a bad block get slot -1, which
 * eesd_kv_append and eesd_kv_read skip, and a bad parent counts as -1.  Tokens that no block covers (a block that
 * the program has cut short) are padding: position, slot and row -1, skipped without a status bit. */
int eesd_tree_meta(const EesdTree* tree, int max_batch, int max_seq, int32_t* status, void* stream);

/* RoPE of q and k and the KV append of n_tok packed tokens into layer `layer`, quantising where the
 * cache is 8-bit.  The rounding of q and k is that of eesd_rope_kv_append (in the model dtype); the 8-bit
 * element is the quantised model-dtype element.  qkv [n_tok, (Hq + 2 Hkv) D], tokens ld_qkv elements apart
 * (ld_qkv % 8 == 0); q_out [n_tok, Hq D] receives the rotated q (NULL: in place in qkv).  tok_pos indexes the
 * RoPE tables [rope_len, D], tok_slot (NULL: tok_pos) the cache.  A token whose position, row or slot is
 * out of range sets a bit in *status and is skipped (all three -1, padding: skipped without).  Two tokens with the same row and slot: the slot
 * holds neither reliably. */
int eesd_kv_append(int dtype, const EesdKvCache* cache, int layer, void* qkv, int ld_qkv, int n_heads,
                   const int32_t* tok_pos, const int32_t* tok_slot, const int32_t* tok_row, int n_tok,
                   const float* rope_cos, const float* rope_sin, int rope_len, void* q_out, int32_t* status, void* stream);

/* k_out / v_out [n_tok, Hkv, D] (each nullable, 16-byte aligned) = the values of layer `layer` at
 * (tok_row[t], tok_slot[t]), in dtype.  A token out of range sets a bit in *status (row and slot -1, padding: none); its outputs are left. */
int eesd_kv_read(int dtype, const EesdKvCache* cache, int layer, const int32_t* tok_slot, const int32_t* tok_row, int n_tok,
                 void* k_out, void* v_out, int32_t* status, void* stream);

/* Attention of tree nodes (or causal chains of any length, e.g. prefill chunks) over one layer of the
 * cache, which already holds the nodes' K and V: node i of a block sees the slots below ctx and those
 * nodes of its block that the mask (NULL: causality) shows; softmax scale 1 / sqrt(D).  A node that sees
 * nothing (ctx 0, empty mask row) gets zeros.  K and V in slots that a node does not see, NaN and
 * infinities among them, do not reach it.  q: rotated queries, tokens ld_q elements apart (ld_q % 8 == 0,
 * 16-byte aligned), Hq D used; out [n_tokens, Hq D].  split_keys: 0 lets the library split long key ranges
 * over CTAs as the launch needs; a multiple of 256 fixes the split, so that a block's result does not
 * depend on the other blocks of the launch (at the same max_nodes, which decides the kernel, and over 8 bits
 * with a mask in both launches or in neither).  workspace:
 * eesd_attn_tree_workspace_bytes() bytes, 256-byte aligned, not initialised, not shared by calls that may
 * overlap.  A block that does not fit the tree's maxima or the cache sets a bit in *status and is skipped.
 * The same call gives the same bits again; what a node does not see does not change a bit of its row.
 * Range: sums of unnormalised weights (up to 2^8 each) and values are held in fp32, and over 8-bit caches q in
 * f16 beside its row's power of two: |q| and, over EESD_KV_MODEL, |V| up to 2^100 stay in range (scores beyond fp32 do not).
 * The weights' roundings, over 8 bits to f16, are relative to the row's largest weight x scale of V. */
size_t eesd_attn_tree_workspace_bytes(int dtype, const EesdKvCache* cache, const EesdTree* tree, int n_heads, int split_keys);
int eesd_attn_tree(int dtype, const EesdKvCache* cache, int layer, const EesdTree* tree, const void* q, int ld_q,
                   int n_heads, void* out, int split_keys, void* workspace, size_t workspace_bytes, int32_t* status,
                   void* stream);

/* Greedy acceptance in a tree (for chains what eesd_greedy_accept computes).  ids[n_tokens]: the node's
 * token; y [n_tokens]: the model's token after the node.  From node 0: go to the lowest-numbered child whose
 * id is y of the current node, until there is none.  path [n_blocks, max_nodes]: the visited nodes, node 0
 * first, then -1; n_acc [n_blocks]: visited nodes - 1; next [n_blocks]: y of the last one.  tree: blk, parent,
 * max_nodes are used.  A bad block sets a bit in *status: path -1, n_acc -1, next -1. */
int eesd_tree_accept(const int32_t* y, const int32_t* ids, const EesdTree* tree, int32_t* path, int32_t* n_acc,
                     int32_t* next, int32_t* status, void* stream);

/* In all layers: slot ctx + j of every block's row = slot ctx + path[b, j], j = 1 .. n_acc[b] (K, V and
 * exponents).  path [n_blocks, max_nodes] must rise (eesd_tree_accept's does); a block whose path does not,
 * or that does not fit, sets a bit in *status and is left as it is, and so are blocks of one row whose slots
 * (ctx .. ctx + T - 1) overlap. */
int eesd_kv_compact(int dtype, const EesdKvCache* cache, const EesdTree* tree, const int32_t* path, const int32_t* n_acc,
                    int32_t* status, void* stream);

/* Device status word helpers for the primitive kernels (a caller-owned int32). */
int eesd_status_read(const int32_t* status, int* bits_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EESD_H */
