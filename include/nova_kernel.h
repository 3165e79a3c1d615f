/*
 * nova_kernel.h -- kernel-layer entry points of the paged KV-cache path (C ABI).
 *
 * One shared library per model geometry (libnova_hip_<model>.so), exactly as
 * the reference welds NH / NKV / HD / L and the page size at compile time
 * (include/nova/model/select.h:6-32, code/graph/kv_pool_cfg.h:12-33): there is
 * no runtime shape argument.  nova_model_geometry() reports what a library was
 * built for.
 *
 * Pool layout (unchanged from the reference, include/nova/model.h:140-145,
 * code/graph/kv_pool.h:8-15): separate K and V pools, each
 *     pool[layer][NB][KB][NKV][HD],  KB = 16 tokens per page,
 * address of token pos of a session = ((layer*NB + table[pos>>4])*KB + (pos&15))*NKV*HD.
 * K/V elements are IEEE fp16 bit patterns (uint16_t); the reference stores fp32
 * (dense.h:25-26), the build stores fp16.  Q and O stay fp32.
 *
 * All launches are asynchronous on the given stream and return nothing; bad
 * arguments abort before anything is launched (include/nova/config.h:42-63).
 */
#ifndef NOVA_KERNEL_H
#define NOVA_KERNEL_H
#include <stddef.h>
#include <stdint.h>
#include "hal.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Geometry the library was compiled for.  Not a reference surface: the
 * reference reads it from ActiveModel (select.h); an FFI needs it as a call. */
typedef struct {
    int nh, nkv, hd, n_layers, kv_block, max_split;
    const char* name;
} nova_geometry;
nova_geometry nova_model_geometry(void);

/* Append n tokens of K and V at logical positions pos0..pos0+n-1.
 * k, v: [n][NKV][HD] fp16.  table: the session's device block table.
 * Replaces nova::launch_kv_store_paged, include/nova/kernel.h:44-45
 * (kernel src/kernel/elem.cu:59-76, launcher :93-98). */
void launch_kv_store_paged(uint16_t* pool_k, uint16_t* pool_v, const int32_t* table, int layer, int nb,
                           int n, int64_t pos0, const uint16_t* k, const uint16_t* v, nova_stream_t s);

/* Single-session split-K decode over keys [0, n_keys) of one layer.
 * q, o: [NH][HD] fp32.  scratch: caller-owned, >= NH*32*(HD+2) floats
 * (src/model.cpp:114,148).  Replaces nova::launch_attn_decode_paged,
 * include/nova/kernel.h:62-64 (attn.cu:197-289 + combine :163-191, launcher :498-512). */
void launch_attn_decode_paged(const float* q, const uint16_t* pool_k, const uint16_t* pool_v,
                              const int32_t* table, int layer, int nb, int n_keys,
                              float* o, float* scratch, nova_stream_t s);

/* Causal attention of n_q new queries at positions n_past..n_past+n_q-1 over
 * keys [0, n_past+qi] (the chunk must already be appended).  q, o:
 * [n_q][NH][HD] fp32.  Replaces nova::launch_attn_prefill_paged,
 * include/nova/kernel.h:65-67 (attn.cu:293-357, launcher :514-525). */
void launch_attn_prefill_paged(const float* q, const uint16_t* pool_k, const uint16_t* pool_v,
                               const int32_t* table, int layer, int nb,
                               int n_q, int n_past, float* o, nova_stream_t s);

/* ---------------- extensions (no single reference counterpart) ---------------- */

/* Batched ragged decode: one launch for all sessions of a layer, optionally
 * fused with that layer's 1-token append.  Replaces the 2N per-session
 * launches of Engine::decode_batch (src/model.cpp:282-289).
 *   q, o     [n_sess][NH][HD] fp32
 *   tables   session i's block table is tables + i*table_stride (the
 *            reference keeps all tables in one array, model.cpp:95)
 *   n_keys   device int32[n_sess]; keys [0, n_keys[i]) are attended
 *   k_new, v_new  NULL, or [n_sess][NKV][HD] fp16: the token at position
 *            n_keys[i]-1 is written into the pool AND attended from these
 *            buffers in the same launch (append-then-attend, dense.h:75-95)
 *   workspace    from attn_decode_batch_workspace_bytes(): plan + split
 *            partials; no initial contents required.
 * Three launches on s: plan, split kernel, combine kernel.
 * n_keys[i] == 0 yields a zero output row. */
size_t attn_decode_batch_workspace_bytes(int n_sess);
/* Status word of the batched decode in `workspace` (n_sess as in the calls):
 * 0, or an OR of failure bits set by the layers since the step's plan launch
 * (1: a split workgroup's in-LDS partial exchange gave up waiting, and the
 * heads it served were written as NaN).  The plan launch clears it.  Waits for
 * the device to finish, then reads the word: a host-side check for tests and
 * serving loops, not for the hot path. */
int attn_decode_batch_status(const void* workspace, int n_sess);
/* The batched call above = launch_attn_decode_plan + launch_attn_decode_paged_planned.
 * A decode step has the same n_keys and block tables in every layer, so a
 * caller can plan once per step and run only the planned call per layer:
 * the plan records each workgroup's session, page range, physical pages and
 * partial slot (a session's workgroups are grouped on one or two XCDs) and
 * the (session, head) each combine block merges (on its session's XCD where
 * there is room), and the planned call starts from one load instead of a dependent
 * n_keys -> partition -> block-table chain.  The plan lives at the start of
 * `workspace`; it is valid until n_keys or the tables change. */
void launch_attn_decode_plan(const int32_t* tables, int table_stride, const int32_t* n_keys, int n_sess,
                             void* workspace, nova_stream_t s);
void launch_attn_decode_paged_planned(const float* q, uint16_t* pool_k, uint16_t* pool_v, const int32_t* tables,
                                      int table_stride, int n_sess, int layer, int nb, const uint16_t* k_new,
                                      const uint16_t* v_new, float* o, void* workspace, nova_stream_t s);
void launch_attn_decode_paged_batch(const float* q, uint16_t* pool_k, uint16_t* pool_v,
                                    const int32_t* tables, int table_stride, const int32_t* n_keys,
                                    int n_sess, int layer, int nb,
                                    const uint16_t* k_new, const uint16_t* v_new,
                                    float* o, void* workspace, nova_stream_t s);
/* The batched decode above (plan + split + combine) with no workspace
 * argument and no allocation: the plan and partials live in a static device
 * array inside the library (about 10 MB per device, held until the process
 * ends).  No counterpart in the reference: it is for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  Limits: n_sess <= 64 on a device of at most 256
 * CUs; anything else aborts with a message before launching.  Every call on
 * a device shares the array, so calls that overlap on one device (two
 * streams) race; calls in one stream order are safe.  Nothing in the array
 * needs clearing between calls. */
void launch_attn_decode_paged_batch_noalloc(const float* q, uint16_t* pool_k, uint16_t* pool_v,
                                            const int32_t* tables, int table_stride, const int32_t* n_keys,
                                            int n_sess, int layer, int nb, const uint16_t* k_new,
                                            const uint16_t* v_new, float* o, nova_stream_t s);
/* The batched decode with the step before it fused in: RopeKvOp
 * (code/graph/dense.h:75-83: rope_batch of q and k at position n_keys[i]-1,
 * src/kernel/rope.cu:21-58, then kv_store_paged of k and v) and the
 * attention of the planned call above, in one launch pair.  k_new, v_new:
 * the layer's new token, fp32 [n_sess][NKV][HD], unrotated; k is rotated with
 * the cs/sn table rows of launch_rope_table (every row used must exist) and
 * written with v as fp16 (nearest even) into the session's last page; q is
 * rotated in registers as it is loaded and the caller's q is not modified.
 * The appended rows are bit-identical to launch_rope_kv_store_paged_batch's;
 * n_keys[i] counts the new token and must be >= 1 for every session. */
void launch_attn_decode_paged_rope_planned(const float* q, const float* k_new, const float* v_new, const float* cs,
                                           const float* sn, uint16_t* pool_k, uint16_t* pool_v,
                                           const int32_t* tables, int table_stride, int n_sess, int layer, int nb,
                                           float* o, void* workspace, nova_stream_t s);
void launch_attn_decode_paged_rope_batch(const float* q, const float* k_new, const float* v_new, const float* cs,
                                         const float* sn, uint16_t* pool_k, uint16_t* pool_v,
                                         const int32_t* tables, int table_stride, const int32_t* n_keys,
                                         int n_sess, int layer, int nb, float* o, void* workspace,
                                         nova_stream_t s);

/* Batched decode in ONE launch for short contexts ("solo"): one workgroup
 * per (kv head, session) streams all of the session's pages for that head,
 * merges its waves on chip and writes the session's output rows itself: no
 * plan, no partials, no combine launch, no workspace.  Arguments as for
 * launch_attn_decode_paged_batch (k_new, v_new: NULL or the fused 1-token
 * append), except that `tables` must hold n_sess full rows of table_stride
 * readable entries (the first min(128, table_stride) entries of a row are read
 * before its n_keys is known).  One CU serves a session's kv head, so this
 * suits steps whose sessions hold up to about 40 pages (640 tokens); longer
 * sessions belong on the split path (on config 1's single 1025-key session
 * the split path is faster).  The reference's launch_attn_decode_paged takes
 * this route itself for contexts up to 24 pages (384 tokens), where it beats
 * that call's own split.  The _rope_ form fuses RoPE
 * as launch_attn_decode_paged_rope_planned does. */
void launch_attn_decode_paged_solo(const float* q, uint16_t* pool_k, uint16_t* pool_v, const int32_t* tables,
                                   int table_stride, const int32_t* n_keys, int n_sess, int layer, int nb,
                                   const uint16_t* k_new, const uint16_t* v_new, float* o, nova_stream_t s);
void launch_attn_decode_paged_rope_solo(const float* q, const float* k_new, const float* v_new, const float* cs,
                                        const float* sn, uint16_t* pool_k, uint16_t* pool_v, const int32_t* tables,
                                        int table_stride, const int32_t* n_keys, int n_sess, int layer, int nb,
                                        float* o, nova_stream_t s);

/* Batched append: session i writes n tokens at positions pos0[i]..pos0[i]+n-1
 * (pos0: device int32[n_sess]) through tables + i*table_stride; k, v:
 * [n_sess][n][NKV][HD] fp16.  One launch for a decode step's appends (or a
 * prefill chunk per session) instead of n_sess launch_kv_store_paged calls. */
void launch_kv_store_paged_batch(uint16_t* pool_k, uint16_t* pool_v, const int32_t* tables, int table_stride,
                                 const int32_t* pos0, int n_sess, int layer, int nb, int n, const uint16_t* k,
                                 const uint16_t* v, nova_stream_t s);

/* Batched chunked-prefill attention: n_sess sessions each with a chunk of n_q
 * queries at positions n_past[i]..n_past[i]+n_q-1 (device int32[n_sess]).
 * q, o: [n_sess][n_q][NH][HD] fp32; tables as for the batched decode.  One
 * launch instead of n_sess launch_attn_prefill_paged calls. */
void launch_attn_prefill_paged_batch(const float* q, const uint16_t* pool_k, const uint16_t* pool_v,
                                     const int32_t* tables, int table_stride, const int32_t* n_past,
                                     int n_sess, int n_q, int layer, int nb, float* o, nova_stream_t s);

/* Batched copy-on-write page copy: for every pair c, copy page src[c] to page
 * dst[c] in every layer of both pools (n_layers*2 pages per pair, one launch).
 * src/dst are device int32[n_pairs].  Replaces the 2L cudaMemcpyAsync calls of
 * Engine::cow_guard, src/model.cpp:178-187. */
void launch_kv_cow_copy(uint16_t* pool_k, uint16_t* pool_v, int nb, const int32_t* src,
                        const int32_t* dst, int n_pairs, nova_stream_t s);

/* Apply a batch of COW decisions in one launch: for each op, copy page src to
 * page dst in every layer of both pools, then set tables_dev[table_index] = dst.
 * ops is a HOST array (copied into the launch, 64 ops per kernel), so no
 * staging buffer or host sync is needed: the fused form of cow_guard's
 * 2L+1 copies (src/model.cpp:171-191) for any number of sessions. */
typedef struct { int32_t src, dst; int64_t table_index; } nova_cow_op;
void launch_kv_cow_apply(uint16_t* pool_k, uint16_t* pool_v, int nb, int32_t* tables_dev,
                         const nova_cow_op* ops, int n_ops, nova_stream_t s);

/* Clear pages (all layers, K and V) -- the per-page memsets of
 * SessionManager::create, code/session.h:107-118, as one launch.
 * pages: device int32[n_pages]. */
void launch_kv_zero_pages(uint16_t* pool_k, uint16_t* pool_v, int nb, const int32_t* pages,
                          int n_pages, nova_stream_t s);

/* Update single entries of device block tables: table_dev[idx[c]] = val[c]
 * for c < n (idx/val are device int32).  The H2D table patch of cow_guard
 * (model.cpp:188-190) for a whole batch of COWs. */
void launch_table_patch(int32_t* table_dev, const int32_t* idx, const int32_t* val, int n,
                        nova_stream_t s);

/* ---- RoPE (src/kernel/rope.cu), NeoX pairs (i, i+HD/2) of the Qwen2 family ---- */

/* cos/sin table [4096][HD/2] fp32 (the reference's kCtx rows, config.h:23).
 * Replaces nova::launch_rope_table, include/nova/kernel.h:47 (rope.cu:9-18,69-72).
 * Each float step of the reference recipe is correctly rounded. */
void launch_rope_table(float* cs, float* sn, nova_stream_t s);
/* The same table with `rows` positions, for contexts past the reference's
 * 4096-row table.  Not a reference surface. */
void launch_rope_table_rows(float* cs, float* sn, int rows, nova_stream_t s);
/* Rotate n tokens in place: q [n][NH][HD], k [n][NKV][HD] fp32 at positions
 * pos0..pos0+n-1.  Replaces nova::launch_rope_batch, kernel.h:48 (rope.cu:39-58,74-80). */
void launch_rope_batch(float* q, float* k, int n, int64_t pos0, const float* cs, const float* sn,
                       nova_stream_t s);
/* One token.  Replaces nova::launch_rope, kernel.h:49 (rope.cu:21-37,82-87). */
void launch_rope(float* q, float* k, int64_t pos, const float* cs, const float* sn, nova_stream_t s);
/* RopeKvOp fused (code/graph/dense.h:75-83: rope_batch, then kv_store_paged):
 * rotate q in place; rotate k and append it with v as fp16 at pos0..pos0+n-1
 * through the block table (k, v: [n][NKV][HD] fp32; k's buffer is left as
 * passed).  One launch and no round trip of K through memory. */
void launch_rope_kv_store_paged(float* q, const float* k, const float* v, const float* cs, const float* sn,
                                uint16_t* pool_k, uint16_t* pool_v, const int32_t* table, int layer, int nb,
                                int n, int64_t pos0, nova_stream_t s);
/* Batched form: session i rotates and appends n tokens at n_past[i]..
 * (device int32[n_sess]) through tables + i*table_stride; q [n_sess][n][NH][HD],
 * k, v [n_sess][n][NKV][HD] fp32.  A decode step's RoPE + append for all
 * sessions (n = 1) or a prefill chunk per session, in one launch. */
void launch_rope_kv_store_paged_batch(float* q, const float* k, const float* v, const float* cs,
                                      const float* sn, uint16_t* pool_k, uint16_t* pool_v,
                                      const int32_t* tables, int table_stride, const int32_t* n_past,
                                      int n_sess, int n, int layer, int nb, nova_stream_t s);

/* ---- Q4_K GEMV (src/kernel/q4k_gemv.cu), weights in ggml block_q4_K
 * (include/nova/quant/q4_k.h:19-25: 144 B per 256 weights, row-major,
 * rows x cols/256 blocks), activations as ActQ8 (include/nova/kernel/types.h:24-28)
 * passed as three plain arrays: int8 codes [rows][cols], fp32 scales
 * [rows][cols/32], int32 sums of each 16 codes [rows][cols/16].  The GEMVs
 * read the three activation arrays with 16-byte loads and abort on pointers
 * that are not 16-byte aligned (the reference's ActQ8 buffers come from its
 * arena, which aligns them). ---- */

/* Quantise rows x cols fp32 activations (cols % 32 == 0).  Replaces
 * nova::launch_quant / launch_quant_ffn, q4k_gemv.cu:196-207 (kernel :9-33),
 * which fix cols to D or FFN at compile time. */
void launch_quant_q8(int8_t* qs, float* d, int32_t* sums, const float* x, int rows, int cols, nova_stream_t s);
/* out[r] = row r of the Q4_K matrix . the quantised activation (one token),
 * cols % 256 == 0, cols <= 32768.  Replaces nova::launch_gemv<K, R>,
 * q4k_gemv.cu:209-213 (kernel :35-91; Q4KWeight = {blocks, rows, cols},
 * types.h:17-21, passed here as plain arguments). */
void launch_gemv_q4k(const uint8_t* blocks, int64_t rows, int cols, const int8_t* xq, const float* xd,
                     const int32_t* xs, float* out, nova_stream_t s);
/* Four tokens: out[t][r] = row r . activation t for t = 0..3 -- the reference's
 * launch_gemv4<K, R> (q4k_gemv.cu:182-187, kernel :98-180), which
 * Engine::decode_batch uses for every projection (model.cpp:270-311).  The
 * four ActQ8 activations are stacked: xq [4][cols], xd [4][cols/32],
 * xs [4][cols/16]; out [4][rows].  Each weight is read once for the four
 * tokens; out[t] equals launch_gemv_q4k on token t up to fp32 summation
 * order (the same terms, summed in another order).
 * cols % 256 == 0, cols <= 28672. */
void launch_gemv4_q4k(const uint8_t* blocks, int64_t rows, int cols, const int8_t* xq, const float* xd,
                      const int32_t* xs, float* out, nova_stream_t s);
/* The quantisation and the GEMVs that share one activation in one launch:
 * n_mat (1..4) Q4_K matrices of the same width cols (blocks[m], rows[m],
 * outs[m]; host arrays) against fp32 x, quantised inside the launch with the
 * arithmetic of launch_quant_q8 (same codes, scales and sums, so outs[m] is
 * bit-identical to launch_quant_q8 followed by launch_gemv_q4k per matrix).
 * Replaces the reference's Kernel::quant (include/nova/kernel.h:80-86,
 * kernel q4k_gemv.cu:9-33) followed by gemm_q4k/launch_gemv for each of the
 * q/k/v or gate/up projections (kernel.h:29-34, q4k_gemv.cu:209-213). */
void launch_gemv_q4k_f32(const uint8_t* const* blocks, const int64_t* rows, float* const* outs, int n_mat,
                         int cols, const float* x, nova_stream_t s);

/* ---- 8-bit pages (no reference counterpart) ----
 *
 * A cache at 132 instead of 256 bytes per row of 128 values: int8 codes c with
 * one fp32 scale s per token, kv head and K or V; value = c * s.  One pool
 *     pool[layer][NB][NKV][4224]  (bytes; kv_q8_page_bytes() = NKV * 4224),
 * 16-byte aligned, with the block tables, positions and page ids of the fp16
 * pools (KB = 16 tokens per page).  The record of a page and kv head holds, for
 * token t of the page and dim d:
 *     K code  int8 at (t>>2)*512 + (d>>4)*64 + (t&3)*16 + (d&15)
 *     V code  int8 at 2048 + d*16 + t
 *     K scale fp32 at 4096 + 4t,  V scale fp32 at 4160 + 4t
 * All-zero memory is a page of zeros.
 *
 * Quantiser, per row x of 128 values: s = fp32(max|x| / 127), codes the integers
 * nearest to the exact quotients x / s, ties to even (s at most the largest
 * number whose 127 s is finite).  A row whose s would be
 * below the smallest normal fp32 number is stored as zeros; a row that holds an
 * infinity or a NaN gets the scale NaN and reads back as NaN.
 *
 * Ragged calls: n_rows rows in all, session i owning rows
 * [row_off[i], row_off[i+1]) of the flat arrays (row_off: device int32[n_sess+1],
 * not decreasing, from 0 to at most n_rows), or n_rows / n_sess rows each where
 * row_off is NULL.  A session may have no rows.  Rows behind the last session's
 * are neither read nor written.  tables must hold n_sess rows of table_stride
 * entries; positions past table_stride * 16 are left out (of the RoPE append with
 * their q), a session that starts below 0 is left out, a table entry outside
 * [0, nb) is not written through and reads page 0.  fp32 arrays and pools are
 * read 16 bytes at a time and must be 16-byte aligned. */
size_t kv_q8_page_bytes(void);
/* Append: session i's rows go to positions pos0[i].. (pos0: device
 * int32[n_sess]).  k, v: [n_rows][NKV][HD] fp32.  Tokens of a page that the call
 * does not write keep their codes and scales.  The 8-bit form of
 * launch_kv_store_paged_batch. */
void launch_kv_q8_store_batch(uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                              const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, const float* k,
                              const float* v, nova_stream_t s);
/* RoPE and append in one launch, the 8-bit form of
 * launch_rope_kv_store_paged_batch: q [n_rows][NH][HD] is rotated in place, k is
 * rotated and quantised with v (k's buffer is left as passed).  The values that
 * are quantised and the rotated q have the bits of launch_rope_batch. */
void launch_rope_kv_q8_store_batch(float* q, const float* k, const float* v, const float* cs, const float* sn,
                                   uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* n_past,
                                   const int32_t* row_off, int n_sess, int n_rows, int layer, int nb,
                                   nova_stream_t s);
/* Read back: the values of positions pos0[i].. of each session as fp32
 * [n_rows][NKV][HD], c * s rounded once. */
void launch_kv_q8_load_batch(const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                             const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, float* k, float* v,
                             nova_stream_t s);
/* Decode attention: one query row per session over keys [0, n_keys[i]) (device
 * int32[n_sess]; the new token already appended).  q, o: [n_sess][NH][HD] fp32.
 * n_keys[i] == 0 gives a row of zeros.  Precision, here and in the chunk attention:
 * fp32 over the values code * scale, but for two roundings.  A query is held to
 * 2^-24 of its largest component, and the product of a key's weight and V
 * scale to 2^-30 of the row's largest such product.  Scores have to be finite in
 * fp32.  Keys that a row does not see do not enter it, whatever they hold, but for
 * this: where a session's V scales differ by more than 2^82, rows that only see the
 * small ones may lose bits.  workspace: from
 * attn_decode_q8_workspace_bytes(n_sess), 16-byte aligned, no initial contents;
 * calls that may overlap need one each. */
size_t attn_decode_q8_workspace_bytes(int n_sess);
void launch_attn_decode_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s);
/* Chunk attention: row r of session i sits at position n_past[i] + r and attends
 * keys [0, n_past[i] + r] (the chunk already appended): prefill chunks of unequal
 * lengths, or a few drafted tokens per session behind long contexts.  q, o:
 * [n_rows][NH][HD] fp32, ragged as above.  max_q: no session has more rows (rows
 * past it are left unwritten).  n_past[i] >= 0.  workspace as for the decode,
 * from attn_chunk_q8_workspace_bytes with the same three counts. */
size_t attn_chunk_q8_workspace_bytes(int n_sess, int n_rows, int max_q);
void launch_attn_chunk_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s);
/* launch_kv_cow_apply and launch_kv_zero_pages for 8-bit pages (page ids outside
 * [0, nb) are not cleared).  The copies of one call run side by side: an op whose dst is another op's dst, or any op's
 * src, aborts the call. */
void launch_kv_q8_cow_apply(uint8_t* pool, int nb, int32_t* tables_dev, const nova_cow_op* ops, int n_ops,
                            nova_stream_t s);
void launch_kv_q8_zero_pages(uint8_t* pool, int nb, const int32_t* pages, int n_pages, nova_stream_t s);

/* ---- rows at positions of their own (no reference counterpart) ----
 *
 * The rotation of launch_rope_batch for any configuration: the first rot_dim dims of a
 * head (even, 2..HD) turn in pairs, half of them apart (dims i and i + rot_dim/2; beside = 0)
 * or side by side (2i and 2i + 1; beside = 1), dims from rot_dim on stay; pair i of a
 * row at position p turns by the angle p * freq[i].  y0 = x0*c - x1*s, y1 = x0*s + x1*c,
 * every product rounded (the bits of launch_rope_batch for the same cos and sin). */
enum { NOVA_ROPE_PLAIN = 0, NOVA_ROPE_LINEAR = 1, NOVA_ROPE_BASE = 2, NOVA_ROPE_BY_PARTS = 3 };
typedef struct {
    int rot_dim;           /* turning dims of a head */
    int scaling;           /* NOVA_ROPE_*, for contexts `factor` times as long as the model's */
    double base;           /* freq[i] = base^(-2i/rot_dim) */
    double factor;         /* >= 1; not read by NOVA_ROPE_PLAIN */
    int train_len;         /* BY_PARTS: the model's own context */
    double slow_turns;     /* BY_PARTS: pairs that turn fewer times over train_len are stretched ... */
    double fast_turns;     /* ... and those that turn more often stay; between, linear in the turns */
} nova_rope_cfg;
/* The pairs' rates in fp32 (host array of rot_dim/2; made in 64 bits) and the factor on
 * cos and sin, once per model.  LINEAR: freq / factor.  BASE: base * factor^(rot_dim /
 * (rot_dim - 2)).  BY_PARTS: a pair turns t = train_len * freq / 2 pi times over the model's own
 * context; its rate is freq from fast_turns on, freq / factor up to slow_turns, and between them
 * freq * (k + (1 - k) / factor), k = (t - slow_turns) / (fast_turns - slow_turns): a ramp that is linear
 * in the turns; the magnitude is 0.1 ln(factor) + 1 (else 1).  Returns rot_dim / 2.
 * There are models whose ramp is linear in the pair's index instead, between the rounded indices
 * of the pairs that turn fast_turns and slow_turns times.  Their rates in between are others (base 10^6,
 * 128 dims, train_len 32768, factor 4, turns 1 to 32: by more than 5% in 15 of 64 pairs, by 42% in
 * one).  launch_rope_angles takes any rates and any magnitude, so such a model's program
 * makes its own, and one that goes without the magnitude passes 1. */
int nova_rope_freqs(const nova_rope_cfg* cfg, float* freq, double* magnitude);
/* The angles of a step's rows, for all layers: cs, sn [n_rows][rot_dim/2] =
 * fp32(cos(pos[r] * freq[i]) * magnitude), and sin, in 64 bits before the one rounding; the angle
 * is exact for |pos| < 2^29.  pos: device int32[n_rows]; freq: device. */
void launch_rope_angles(const int32_t* pos, int n_rows, const float* freq, int rot_dim, double magnitude, float* cs,
                        float* sn, nova_stream_t s);
/* Turn q [n_rows][NH][HD] into q_out and k [n_rows][NKV][HD] into k_out (each may be its own
 * input).  Rows whose pos is negative (launch_kv_step_plan's empty rows) are left as they are; pos
 * may be NULL: all rows.  All fp32 arrays 16-byte aligned. */
void launch_rope_rows(const float* q, const float* k, const int32_t* pos, const float* cs, const float* sn, int n_rows,
                      int rot_dim, int beside, float* q_out, float* k_out, nova_stream_t s);

/* ---- 4-bit pages (no reference counterpart) ----
 *
 * A cache at 68 instead of 256 bytes per row of 128 values: 4-bit floating point codes
 * (0, .5, 1, 1.5, 2, 3, 4, 6 for codes 0..7, the sign in bit 3) with a power of two per 32
 * dims, held as its exponent plus 127 in a byte: the block-scaled fp4 operand of the
 * matrix instructions.  One pool
 *     pool[layer][NB][NKV][2176]  (bytes; kv_q4_page_bytes() = NKV * 2176),
 * 16-byte aligned, with the block tables, positions and page ids of the other pools.  The
 * record of a page and kv head holds, for token t of the page and dim d:
 *     K code       at t*64 + (d>>1), the low half of the byte for even d
 *     V code       at 1024 + (d>>5)*256 + (d&15)*16 + t, the low half where bit 4 of d is clear
 *     K exponent   at 2048 + (t&3)*16 + (d>>5)*4 + (t>>2)
 *     V exponent   at 2112 + (d>>5)*16 + t
 * An exponent byte b stands for 2^(b - 127), 255 for NaN; 0 stands beside codes of zero only.  All-zero
 * memory is a page of zeros.
 *
 * Quantiser, per 32 values with largest |x| = a: the power is the smallest 2^e with
 * a <= 7 * 2^e, the codes the values nearest to x / 2^e, ties to the even code, so that no
 * value is off by more than half its step.  e is at most 96 (values past 7 * 2^96 are held as
 * 6 * 2^96); where it would be below -100 the 32 are stored as zeros.  A row of 128 that holds an infinity or a NaN gets the exponent byte 255
 * in all its blocks and reads back as NaN.
 *
 * Ragged calls, tables, positions outside them and alignment are those of the 8-bit calls above. */
size_t kv_q4_page_bytes(void);
/* Append: the 4-bit form of launch_kv_q8_store_batch. */
void launch_kv_q4_store_batch(uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                              const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, const float* k,
                              const float* v, nova_stream_t s);
/* Rotation and append in one launch: q's rows turn into q_out (which may be q), k's rows turn and
 * are quantised with v's (k's buffer is left as passed).  cs, sn: the rows' angles from
 * launch_rope_angles; rot_dim and beside as in launch_rope_rows, whose bits the turned
 * rows have.  Of the 14B shape at most about 13 million rows a call (as many as a launch has
 * threads for), else 2^24 as everywhere. */
void launch_rope_rows_kv_q4_store_batch(const float* q, const float* k, const float* v, const float* cs, const float* sn,
                                        int rot_dim, int beside, uint8_t* pool, const int32_t* tables, int table_stride,
                                        const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int layer,
                                        int nb, float* q_out, nova_stream_t s);
/* Read back as fp32 [n_rows][NKV][HD]; every value is exact. */
void launch_kv_q4_load_batch(const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                             const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, float* k, float* v,
                             nova_stream_t s);
/* Decode and chunk attention: the calls of the 8-bit pages, with the same arguments.
 * Precision: fp32 over the values of the codes, but for two roundings.  A query (times
 * 1/sqrt(HD) log2 e) is held to 2^-24 of the largest of each 32 of its dims, or to 2^-124.  In
 * a tile (64 keys from a multiple of 64) whose V powers of two lie within 2^7 of each other, and from
 * 2^-13 to 2^13, a key's weight is held to 2^-22 of itself, or to 2^-26 of the row's largest weight in that tile, or to 2^-104 of
 * the row's largest; in any other tile it goes in whole.  Scores have to be finite in fp32.  Keys that a
 * row does not see do not enter it, whatever they hold (only, their powers may decide which of the two
 * a tile is). */
size_t attn_decode_q4_workspace_bytes(int n_sess);
void launch_attn_decode_q4_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s);
size_t attn_chunk_q4_workspace_bytes(int n_sess, int n_rows, int max_q);
void launch_attn_chunk_q4_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s);
/* launch_kv_q8_cow_apply and launch_kv_q8_zero_pages for 4-bit pages. */
void launch_kv_q4_cow_apply(uint8_t* pool, int nb, int32_t* tables_dev, const nova_cow_op* ops, int n_ops,
                            nova_stream_t s);
void launch_kv_q4_zero_pages(uint8_t* pool, int nb, const int32_t* pages, int n_pages, nova_stream_t s);

/* ---- a step's bookkeeping on the GPU (no reference counterpart) ----
 *
 * For servers that give sessions their pages as they grow: the pages of a pool that no
 * session holds are a stack on the device (free_pages[0 .. *n_free), room for nb), and one call per
 * step turns the sessions' lengths into everything that the step's calls take.  Any page
 * format; a page belongs to one session (sessions that share pages stay with the session
 * manager of nova_graph.h).
 *
 * Session i holds n_have[i] tokens, keeps the first n_keep[i] of them (n_keep NULL: all; 0: it
 * ends) and adds n_new[i].  With pages(n) = ceil(n / 16):
 *   - its pages [pages(keep), pages(have)) go back: on top of the stack, in (session, page)
 *     order, the first of all on top;
 *   - it takes pages(keep + new) - pages(keep) pages from the top, sessions in order, into its
 *     row of `tables`.  The first session with which the step's rows would pass max_rows
 *     or its pages would pass the free ones gets no rows, nor does any after it; one whose
 *     table is too short for keep + new gets none and the others are served.
 *     Rows stand without gaps: behind a session that got none, the others' stand further up, by
 *     row_off, and not where sums of n_new or the session's index would put them.
 * Lengths below 0 count as 0, n_have past the table as full, n_keep past n_have as n_have.
 * Out (device): n_past[i] = keep, n_keys[i] = keep + rows granted, row_off [n_sess+1] their sums, and
 * for each row r of max_rows its position pos[r] and its place in the cache slots[r] =
 * page * 16 + pos % 16 (-1 where the page is outside [0, nb)); rows behind the last have -1 in both.
 * *n_free_left: pages free afterwards.  n_keys or n_past may be n_have, n_free_left may be n_free; else
 * no output overlaps another array.  pos and slots may be NULL if max_rows is 0.  workspace: 16-byte aligned, no
 * initial contents; calls that may overlap need one each. */
size_t kv_step_plan_workspace_bytes(int n_sess);
void launch_kv_step_plan(int32_t* tables, int table_stride, const int32_t* n_have, const int32_t* n_keep,
                         const int32_t* n_new, int n_sess, int max_rows, int32_t* free_pages, const int32_t* n_free, int nb,
                         int32_t* n_past, int32_t* n_keys, int32_t* row_off, int32_t* pos, int64_t* slots,
                         int32_t* n_free_left, void* workspace, nova_stream_t s);

#ifdef __cplusplus
}
#endif
#endif
