/*
 * tie_hip.h -- C ABI of the MI355X (gfx950) Qwen3-MoE FFN block for TIE.
 *
 * The reference (szemzoa/tie) runs the MoE FFN inline in
 * transformer_layer_qwen3 (model_qwen3.c:404-471): per token a router GEMV
 * (dispatch_mat_vec, model_qwen3.c:431-432), find_top_k (engine.c:891),
 * softmax over the k selected logits (engine.c:864), k process_expert_task
 * jobs on the thread pool (engine.c:916-964) and an fp32 weighted combine
 * (model_qwen3.c:459-470).  This library replaces that whole branch with
 * HIP kernels.  Every entry point is plain C: pointers, sizes and GGML type
 * ids (gguf.h:8-36), no HIP or torch types.
 *
 * Return codes: 0 on success, a negative TIE_HIP_E* code otherwise; the
 * library never exits the process.  tie_hip_last_error() describes the
 * last failure of the calling thread.
 */
#ifndef TIE_HIP_H
#define TIE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TIE_HIP_ABI_VERSION 2

/* GGML type ids as in gguf.h:8-36 */
#define TIE_GGML_F32 0
#define TIE_GGML_F16 1
#define TIE_GGML_Q4_K 12
#define TIE_GGML_Q6_K 14
#define TIE_GGML_I8 24
#define TIE_GGML_BF16 30

#define TIE_HIP_OK 0
#define TIE_HIP_EINVAL (-1)  /* bad argument, shape or type (TIE: return -1, model_qwen3.c:407-410) */
#define TIE_HIP_EHIP (-2)    /* a HIP runtime error */
#define TIE_HIP_ENOMEM (-3)  /* device allocation failed */
#define TIE_HIP_ENOINIT (-4) /* tie_hip_init() not called */

#define TIE_SILU_TABLE_SIZE 8192 /* SILU_TABLE_SIZE, engine.h:10 */

/* Forward flags */
#define TIE_HIP_PATH_AUTO 0x0  /* exact fp32 GEMV path up to tie_hip_exact_max_tokens() (21), 16-bit MFMA grouped GEMM above */
#define TIE_HIP_PATH_EXACT 0x1 /* always the fp32 path that reproduces TIE's arithmetic bit for bit */
#define TIE_HIP_PATH_MFMA 0x2  /* always the grouped-GEMM path */

/* Routing modes (tie_hip_layer_desc.routing) */
#define TIE_HIP_ROUTE_SOFTMAX 0 /* Qwen3: top-k of the logits, softmax over the k (model_qwen3.c:431-443) */
#define TIE_HIP_ROUTE_SIGMOID 1 /* LFM2: sigmoid, top-k of sigmoid + bias, L1-normalised sigmoid of the k
				   (model_lfm2.c:437-467) */

typedef struct tie_hip_layer tie_hip_layer;

/* Library set-up on one HIP device; replaces the MoE-relevant part of
 * engine_alloc (engine.c:14-40: thread pool, silu_table_init,
 * math_dispatch_init).  Builds the SiLU table on the host CPU the way TIE
 * does and uploads it. */
int tie_hip_init(int device);

/* Frees every device resource, including the weight cache. */
void tie_hip_shutdown(void);

/* Text of the last error on the calling thread ("" when none). */
const char *tie_hip_last_error(void);

/* Drop-in for the MoE branch of transformer_layer_qwen3
 * (model_qwen3.c:404-471).  Host pointers, as TIE holds them:
 *   x          ctx->mem.normed_ffn_input, [T][d] F32
 *   router_w   ffn_gate_inp, F32 [E][d] (router_type must be TIE_GGML_F32)
 *   gate/up    ffn_{gate,up}_exps, [E][F][d] in GGUF block layout
 *   down       ffn_down_exps, [E][d][F] in GGUF block layout
 *   out        ctx->mem.ffn_down_output, [T][d] F32
 *   topk_idx_opt / topk_w_opt  optional [T][k] selected experts / weights
 * Expert types: TIE_GGML_Q4_K, TIE_GGML_Q6_K or TIE_GGML_BF16.  d and F must
 * be multiples of 256, k <= E <= 1024, k <= 32.  Weight tensors are uploaded
 * once and cached, keyed by host pointer, type and size (they must stay
 * valid and unchanged while cached, as TIE's mmap'd weights are).  Runs on
 * the library's stream and returns after out is written. */
int tie_hip_moe_ffn(const float *x, int T, int d, int F, int E, int k, const void *router_w, int router_type,
		    const void *gate_exps, int gate_type, const void *up_exps, int up_type, const void *down_exps,
		    int down_type, float *out, int32_t *topk_idx_opt, float *topk_w_opt);

/* Drop-in for the MoE branch of transformer_layer_lfm2
 * (model_lfm2.c:414-497).  Same arguments as tie_hip_moe_ffn plus
 *   probs_bias_opt  exp_probs_b_bias, F32 [E] host array, or NULL (the
 *                   branch at model_lfm2.c:446-454)
 * Routing is TIE_HIP_ROUTE_SIGMOID: p_e = 1/(1+expf(-logit_e)), top-k of
 * p_e + bias_e, weights p_j / (sum_j p_j + 1e-6); the experts and the
 * combine are those of tie_hip_moe_ffn. */
int tie_hip_moe_ffn_lfm2(const float *x, int T, int d, int F, int E, int k, const void *router_w, int router_type,
			 const float *probs_bias_opt, const void *gate_exps, int gate_type, const void *up_exps,
			 int up_type, const void *down_exps, int down_type, float *out, int32_t *topk_idx_opt,
			 float *topk_w_opt);

/* Drop-in for the whole FFN half of transformer_layer_qwen3 (the RMSNorm at
 * model_qwen3.c:392-401, the MoE branch at :404-471 and the residual add at
 * :491): hidden += MoE(rms_norm(hidden, ffn_norm, eps)).
 *   hidden    ctx->mem.hidden_state, [T][d] F32, read and updated in place
 *   ffn_norm  LayerWeights.ffn_norm (engine.h:72), F32 [d]
 *   eps       ctx->model->norm_eps
 * The RMSNorm reproduces rms_norm_f32_f32_f32_avx2 (math_avx2.c:56-96) as
 * TIE's build computes it, including the host CPU's RSQRTSS approximation
 * (tabulated on this host at the first call).  Other arguments as
 * tie_hip_moe_ffn. */
int tie_hip_qwen3_ffn(float *hidden, int T, int d, int F, int E, int k, const float *ffn_norm, float eps,
		      const void *router_w, int router_type, const void *gate_exps, int gate_type, const void *up_exps,
		      int up_type, const void *down_exps, int down_type, int32_t *topk_idx_opt, float *topk_w_opt);

/* Replace the SiLU lookup table with the caller's (TIE's own silu_table,
 * engine.c:12, as filled by silu_table_init, engine.c:297-303). */
int tie_hip_set_silu_table(const float *table, int n);

/* Build the SiLU table on the host CPU exactly as TIE's compiled
 * silu_table_init does on this host (no GPU needed). */
int tie_hip_silu_table_host(float *table, int n);

/* ------------------------------------------------------------------ */
/* Device-resident layers (inputs already in HBM)                       */
/* ------------------------------------------------------------------ */

typedef struct tie_hip_layer_desc {
	int d, F, E;
	const void *router_w; /* F32 [E][d] */
	int router_type;      /* TIE_GGML_F32 */
	const void *gate_exps;
	int gate_type;
	const void *up_exps;
	int up_type;
	const void *down_exps;
	int down_type;
	const float *router_bias; /* optional [E], added to the logits before top-k; NULL in TIE */
	int src_on_device;        /* 1: the pointers above are device memory (GGUF layout); the
				     library drains the device before reading them, so work on any
				     stream that writes them has finished */
	int literal_bf16_stride;  /* 1: BF16 experts start at e*rows*(in/256)*2 bytes, as
				     process_expert_task computes it (engine.c:929-942) */
	int routing;              /* TIE_HIP_ROUTE_SOFTMAX (0, Qwen3) or TIE_HIP_ROUTE_SIGMOID (LFM2) */
	const float *probs_bias;  /* optional [E]: LFM2's exp_probs_b_bias, added to the sigmoid
				     scores for the selection only (ROUTE_SIGMOID) */
} tie_hip_layer_desc;

/* Upload (or copy on device) and repack one layer's weights into the
 * device layout.  The source buffers may be freed afterwards.  With
 * src_on_device (and for tie_hip_matrix_create likewise) the library drains
 * the device (hipDeviceSynchronize): no thread may be capturing a HIP graph
 * meanwhile, as a device synchronisation fails or invalidates a capture in
 * global or relaxed mode. */
int tie_hip_layer_create(const tie_hip_layer_desc *desc, tie_hip_layer **out);
void tie_hip_layer_destroy(tie_hip_layer *layer);

/* Device bytes held by a layer. */
size_t tie_hip_layer_bytes(const tie_hip_layer *layer);

/* Every call on device pointers is enqueued on its `stream`: a hipStream_t,
 * NULL for the library's stream (non-blocking: it is ordered with no other
 * stream, the default one among them), or this for HIP's default stream,
 * whose handle is 0. */
#define TIE_HIP_STREAM_DEFAULT ((void *)1)

/* MoE block on device pointers, enqueued on `stream` (a hipStream_t; NULL =
 * the library stream).  x_dev/out_dev are [T][d] F32; topk outputs are
 * optional [T][k].  Returns once enqueued; the caller synchronises.
 *
 * Streams: the library keeps one scratch workspace per stream, so forwards
 * enqueued on different streams never share scratch memory and may run
 * concurrently (on distinct out buffers; the topk buffers are only written,
 * so sharing them spoils them alone).  Forwards on one stream are
 * ordered by that stream.  When a call needs a larger workspace than its
 * stream holds, the library drains the whole device (hipDeviceSynchronize)
 * before freeing the old one; a call made during HIP graph capture must
 * therefore not grow it (warm the stream up with the largest T first).
 *
 * One token (T = 1, eager) runs as one launch whose workgroups hand values
 * to each other; their waits are bounded.  Should a wait give up (the GPU
 * did not run the workgroups together, e.g. under heavy sharing), that
 * call's outputs are NaN and the stream's status word is set: the
 * synchronous entry points (tie_hip_moe_ffn, _lfm2, tie_hip_qwen3_ffn)
 * then return TIE_HIP_EHIP, and device-API callers read it with
 * tie_hip_stream_status. */
/* Frees the scratch workspace the library keeps for `stream` (grown by the
 * forwards enqueued on it; at the 235B shape and large T, hundreds of MiB).
 * Call it before destroying a stream that forwards ran on; otherwise the
 * workspace lives until tie_hip_shutdown.  Drains the device first.  A graph
 * captured with that workspace is not to be replayed afterwards. */
int tie_hip_stream_release(void *stream);

int tie_hip_moe_forward(tie_hip_layer *layer, const float *x_dev, int T, int k, float *out_dev,
			int32_t *topk_idx_dev, float *topk_w_dev, int flags, void *stream);

/* tie_hip_moe_forward that allocates nothing: no counterpart in the
 * reference.  For callers that cannot allocate device memory (code under
 * HIP graph capture, serving loops, harnesses that forbid hipMalloc).  Its
 * scratch is one static 24 MiB device array per GPU (held until the process
 * ends) instead of the per-stream workspace: calls whose scratch would not
 * fit (T * k pairs with this layer's shape: T <= 89 at d = 2048, F = 768,
 * k = 8; T <= 44 at d = 4096, F = 1536, k = 8) return TIE_HIP_EINVAL.  All calls on a GPU share the array,
 * so calls that overlap in time on one GPU (other streams, other threads)
 * race: serialise them.  Same arguments, results and stream rules as
 * tie_hip_moe_forward otherwise. */
int tie_hip_moe_forward_noalloc(tie_hip_layer *layer, const float *x_dev, int T, int k, float *out_dev,
				int32_t *topk_idx_dev, float *topk_w_dev, int flags, void *stream);

/* The same FFN half on device pointers: out_dev = hidden_dev +
 * block(rms_norm(hidden_dev)), both [T][d] F32; out_dev may be hidden_dev
 * (TIE's in-place update).  ffn_norm_dev [d] F32.  Enqueued on `stream` like
 * tie_hip_moe_forward. */
int tie_hip_moe_forward_residual(tie_hip_layer *layer, const float *hidden_dev, const float *ffn_norm_dev, float eps,
				 int T, int k, float *out_dev, int32_t *topk_idx_dev, float *topk_w_dev, int flags,
				 void *stream);

/* ------------------------------------------------------------------ */
/* Dense matrices (dispatch_mat_mat with F32 input)                     */
/* ------------------------------------------------------------------ */

typedef struct tie_hip_matrix tie_hip_matrix;

/* Upload one GGUF weight matrix [rows][in_dim] (ne = [in_dim, rows]) of type
 * TIE_GGML_F32, Q4_K, Q6_K or BF16 (repacked into the panel layout); rows a
 * multiple of 64, in_dim a multiple of 256 up to 16384.  The source may be
 * freed afterwards. */
int tie_hip_matrix_create(const void *w, int type, int rows, int in_dim, int src_on_device, tie_hip_matrix **out);
void tie_hip_matrix_destroy(tie_hip_matrix *m);

/* dispatch_mat_mat (math_dispatch.c:304-359) on device pointers:
 * out_dev[t][r] = W[r] . x_dev[t] for t < T, x [T][in_dim] F32, out
 * [T][rows] F32.  TIE_HIP_PATH_EXACT and TIE_HIP_PATH_AUTO (the default, at
 * every T) use TIE's row kernels (mat_vec_row_f32_{f32,q4k,q6k,
 * bf16}_f32_avx2) bit for bit.  TIE_HIP_PATH_MFMA (opt-in; Q4_K or Q6_K,
 * rows a multiple of 256) runs the f16 matrix cores with fp32 accumulation
 * (relative L2 error about 3e-4 of TIE's result); rows whose input does not
 * fit the f16 range are recomputed with the exact kernel.
 * TIE_HIP_PATH_MFMA on an unsupported matrix is an error.  Enqueued on `stream`.  The attention projections, the dense FFN and the LM
 * head of transformer_layer_qwen3 / main.c use it. */
int tie_hip_mat_mat(tie_hip_matrix *m, const float *x_dev, int T, float *out_dev, int flags, void *stream);

/* ------------------------------------------------------------------ */
/* The attention half for drafted tokens: a paged key/value cache        */
/* ------------------------------------------------------------------ */
/* What lies between a layer's projections (tie_hip_mat_mat) and its FFN half
 * (tie_hip_moe_forward_residual), and behind the LM head: the norms of queries
 * and keys for each head, the rotation and the cache write (tie_hip_kv_append),
 * the attention of a tree of drafted tokens, a prompt's chunk or single tokens
 * (tie_hip_tree_attention), the accepted path (tie_hip_verify_tree) and its
 * rows (tie_hip_kv_keep).  Everything is on device pointers, enqueued on
 * `stream` (NULL: the library stream) and captures into HIP graphs.  No call
 * here reproduces TIE's arithmetic bit for bit: they are held to 64-bit
 * results (F32 outputs to about 1e-6 relative; an element of the attention's to
 * that of sum_j p_j max_i |v_ji|, the rows' largest magnitudes by their weights;
 * over f16 rows, weights below 2^-36 of the largest may be taken for 0).
 *
 * The caller owns the cache's memory, in pages of TIE_HIP_PAGE_ROWS rows (a
 * row: one token) that the layers share the numbering of:
 *   k  [n_layers][n_pages][kv_heads][64][head_dim]
 *   v  [n_layers][n_pages][kv_heads][head_dim][64]
 * as f16, or as int8 codes with F32 scales [n_layers][n_pages][kv_heads][64]
 * (value = code * scale; scale = largest magnitude of the row's head / 127,
 * code = the nearest whole number to value / scale, ties to even).  Values
 * beyond the f16 range are held as the largest f16; an int8 row with a value
 * that is not finite has scale NaN.  Pages need no clearing. */
#define TIE_HIP_PAGE_ROWS 64

typedef struct tie_hip_kv_cache {
	int type;     /* TIE_GGML_F16 or TIE_GGML_I8 */
	int n_layers; /* layers in the arrays */
	int n_pages;  /* pages of a layer, at most 2^25 */
	int kv_heads;
	int head_dim; /* 64 or 128 */
	void *k, *v;  /* 16-byte aligned */
	float *k_scale, *v_scale; /* TIE_GGML_I8; else NULL */
} tie_hip_kv_cache;

/* The sequences of a call, as device arrays.  Sequence b has `len[b]` rows in
 * the cache (committed: every token of it sees them) and the token rows
 * first[b] .. first[b + 1] - 1 of the activations; its token j is cache row
 * len[b] + j, on page pages[b][(len[b] + j) / 64].  Rows that belong to no
 * sequence are left as they are.  The arrays are read on the device, so no call
 * can refuse what they say; it is checked there.  Where a sequence's rows do not
 * lie within its row of the page table (a length below 0 or too large), or one's
 * page is none, nothing is written to the cache for them, and the outputs that
 * would need them are NaN (of the attention others of the sequence may be, too).
 * A sequence whose range of token rows falls, begins below 0 or ends past
 * n_tokens has no rows in the call.  Where ranges that do not ascend overlap, a row's outputs
 * are those of one of its sequences, and its cache row is written for one at
 * most.  (tie_hip_verify_tree: where any range does not ascend within the rows,
 * no sequence has any.) */
typedef struct tie_hip_kv_seqs {
	int n_seqs;           /* at most 65535 */
	int max_pages;        /* columns of the page table */
	int n_tokens;         /* token rows of the activations */
	const int32_t *pages; /* [n_seqs][max_pages] */
	const int32_t *len;   /* [n_seqs] */
	const int32_t *first; /* [n_seqs + 1], ascending; NULL: one token for each sequence */
} tie_hip_kv_seqs;

/* Norm, rotation and cache write of the sequences' tokens in one layer, one
 * launch.  q, k, v: F32 rows of the projections, `*_stride` floats from a
 * token to the next (all three may lie in one matrix); q has n_heads heads (a
 * multiple of kv_heads), k and v kv_heads.
 *   norm      x * w / sqrt(mean(x^2) + eps) over each head, q_norm and k_norm
 *             F32 [head_dim] (NULL: none)
 *   rotation  the pair (x[i], x[i + head_dim / 2]) by pos * theta^(-2 i /
 *             head_dim); pos [n_tokens] (a tree's nodes at one depth share a
 *             position), NULL: the token's cache row (a query without one, as
 *             its sequence's length is none, is NaN)
 * in 64 bits, rounded once.  The queries go to q_out (which may be q, with the
 * same stride, or other columns of the same matrix; it shares no memory with k, v,
 * pos or the sequences' arrays), keys and values to the cache. */
int tie_hip_kv_append(const tie_hip_kv_cache *cache, int layer, const tie_hip_kv_seqs *seqs, const float *q, size_t q_stride,
		      const float *k, size_t k_stride, const float *v, size_t v_stride, int n_heads, const float *q_norm,
		      const float *k_norm, float eps, float theta, const int32_t *pos, float *q_out, size_t q_out_stride,
		      void *stream);

/* tie_hip_kv_append for tokens whose position has several axes (time, height
 * and width of an image's patches): pair i is rotated by pos[axis[i]][t] *
 * theta^(-2 i / head_dim).
 *   pos   [n_axes][n_tokens] (text has the same position on all axes)
 *   axis  [head_dim / 2], each below n_axes: host memory, read before the call
 *         returns (a captured graph keeps what it said)
 * Positions need not be cache rows: an image's tokens take fewer positions than
 * rows, and a cache's rows, masks and windows go by rows. */
#define TIE_HIP_MAX_AXES 4
int tie_hip_kv_append_axes(const tie_hip_kv_cache *cache, int layer, const tie_hip_kv_seqs *seqs, const float *q,
			   size_t q_stride, const float *k, size_t k_stride, const float *v, size_t v_stride, int n_heads,
			   const float *q_norm, const float *k_norm, float eps, float theta, const int32_t *pos, int n_axes,
			   const uint8_t *axis, float *q_out, size_t q_out_stride, void *stream);

/* The cache rows of the sequences' tokens as F32, of n_layers layers from
 * `layer` on: k_out and v_out [n_layers][n_tokens][kv_heads][head_dim].  (len
 * of zeros and first over whole lengths reads whole sequences.) */
int tie_hip_kv_read(const tie_hip_kv_cache *cache, int layer, int n_layers, const tie_hip_kv_seqs *seqs, float *k_out,
		    float *v_out, void *stream);

/* Attention of the sequences' tokens over their committed rows and, of their
 * own tokens, those that `mask` names: bit j % 64 of mask[t][j / 64] says that
 * token row t sees token j of its sequence ([n_tokens][mask_words]; tokens past
 * the words are not seen).  mask NULL: token i sees tokens 0 .. i (a prompt's
 * chunk, a chain, a single token).  A row that sees nothing gives 0.
 *   q    [n_tokens] rows of n_heads heads (as tie_hip_kv_append leaves them)
 *   out  the same shape (may be q, with the same stride; it shares no memory with
 *        the mask or the sequences' arrays)
 *   work work_bytes of device memory, 16-byte aligned, at least
 *        tie_hip_tree_attention_work_bytes, filled with zeros before the first
 *        call that gets it and after anything else has written to it (calls
 *        here leave it fit for the next); what is enough for a call is enough
 *        for every one of the same heads and cache type with no more tokens,
 *        sequences and columns of the page table.  NULL: the stream's
 *        workspace, which all calls on the stream share and which grows as
 *        needed, but not during HIP graph capture (run the largest call once
 *        before, on the stream that captures, or pass memory).  Calls and
 *        graphs that may run at the same time on different streams need memory
 *        of their own.
 * Scores are held in F32; past 2^24 in magnitude their rounding is larger than
 * what a softmax tells apart, and a row's result means nothing.
 * A row's result is the same whatever else the call holds only up to F32
 * rounding: which kernel takes the rows and how they are cut follows the
 * lengths and the call's sizes, the page table's columns among them.  Two equal
 * calls give equal bits.  A value in the cache that is not finite does nothing
 * to the results that do not see its row; of those that do it spoils its column
 * (an f16 value of V) or all of the head's (a key or a scale). */
size_t tie_hip_tree_attention_work_bytes(const tie_hip_kv_cache *cache, const tie_hip_kv_seqs *seqs, int n_heads);
int tie_hip_tree_attention(const tie_hip_kv_cache *cache, int layer, const tie_hip_kv_seqs *seqs, const float *q,
			   size_t q_stride, int n_heads, float scale, const uint64_t *mask, int mask_words, float *out,
			   size_t out_stride, void *work, size_t work_bytes, void *stream);

/* tie_hip_tree_attention through a sliding window, with a few first rows that
 * stay visible: token t of a sequence, which stands at row at[t] ([n_tokens];
 * NULL: its own row, len + its index), sees row r of the committed ones where
 *   r < sinks  or  r > at[t] - window
 * (at says where a window begins, not where it ends: all committed rows above
 * are seen).  mask NULL: its own tokens up to itself, by the same rule for their
 * rows.  With a mask: the own tokens that it names, whatever the window.  A tree
 * of drafted tokens has at = len + the node's depth, and no bits for ancestors
 * that lie behind the window.
 * Pages that hold no row that a token sees are not looked at: their entries in
 * the page table may be none, as tie_hip_kv_plan leaves them.
 * window at least 1, sinks 0 or more; out shares no memory with at either; everything
 * else, scratch memory included, as for tie_hip_tree_attention.  The work bytes are enough for any window. */
size_t tie_hip_window_attention_work_bytes(const tie_hip_kv_cache *cache, const tie_hip_kv_seqs *seqs, int n_heads);
int tie_hip_window_attention(const tie_hip_kv_cache *cache, int layer, const tie_hip_kv_seqs *seqs, const float *q,
			     size_t q_stride, int n_heads, float scale, int window, int sinks, const int32_t *at,
			     const uint64_t *mask, int mask_words, float *out, size_t out_stride, void *work, size_t work_bytes,
			     void *stream);

/* Keep the accepted path of each sequence: cache row len + path[b][j] becomes
 * row len + j for j < n_keep[b], in all layers, and len_out[b] = len[b] +
 * n_keep[b] (len_out may be len; NULL: not wanted).  path [n_seqs][max_path]
 * holds tokens of the sequence, ascending; an entry that does not ascend, is
 * no token of it, or whose row lies on no page, before or after, ends the path
 * there. */
int tie_hip_kv_keep(const tie_hip_kv_cache *cache, const tie_hip_kv_seqs *seqs, const int32_t *path, int max_path,
		    const int32_t *n_keep, int32_t *len_out, void *stream);

/* The pages of a step, from the requests' lengths: one row of the page table
 * for each request, pages taken from a pool of free ones and given back to it, and
 * where the step's tokens go.  Everything is on the device, so that a captured
 * graph goes on while requests grow.
 *
 * The pool: free pages lie in a ring, free[state[0]], free[state[0] + 1], ...
 * (after the last place the first), state[1] of them.  Pages are taken from its head;
 * pages that come free are put behind its tail, and can be had from the next
 * call on.  A state that is none (a place outside the ring, more than n_pages) has
 * no pages and takes none.
 *
 * Request b has len[b] rows and asks for n_new[b] more; its pages in
 * ceil(len / 64) .. ceil((len + n_new) / 64) - 1 that the table does not name are
 * taken from the pool (a page that an earlier call's drafts left there stays).
 * Requests are served in order: the first whose pages or token rows are not
 * there any more and all behind it get nothing (first[b + 1] = first[b]).  One whose
 * rows do not lie within its row of the table (len below 0, or too large) asks for
 * nothing.  n_new below 0: the request has ended, and all its pages go back.
 * window > 0: of every other request the pages go back that the next token, at
 * row len, and those after it do not see through tie_hip_window_attention: those whose
 * rows all lie below len - window + 1, but for those of the first `sinks` rows.  Entries
 * of pages that went back are -1.  Where more pages come back than the ring has
 * places (a page named twice), those left over stay in the table.
 *   pages      [n_seqs][max_pages]; pages_out the same shape, the new table (may be pages)
 *   first      [n_seqs + 1] the requests' token rows: tie_hip_kv_seqs.first
 *   pos, slot  [n_tokens] or NULL: each token row's place in its sequence (its
 *              cache row), and in the cache (page * 64 + row in it); -1 for rows
 *              of no request and (slot) rows on no page
 *   state_out  the pool's state behind the call (may be state)
 * n_tokens is the most token rows that the step has.  No other output may share
 * memory with an input or another output.  work as for tie_hip_tree_attention. */
typedef struct tie_hip_kv_pool {
	int n_pages;          /* of a layer of the cache */
	int32_t *free;        /* [n_pages] */
	const int32_t *state; /* [2] */
	int32_t *state_out;   /* [2] */
} tie_hip_kv_pool;

size_t tie_hip_kv_plan_work_bytes(int n_seqs);
int tie_hip_kv_plan(const tie_hip_kv_pool *pool, int n_seqs, int max_pages, int n_tokens, const int32_t *pages,
		    const int32_t *len, const int32_t *n_new, int window, int sinks, int32_t *pages_out, int32_t *first,
		    int32_t *pos, int32_t *slot, void *work, size_t work_bytes, void *stream);

/* Log-probabilities under p = softmax(logits / temperature) of each row:
 *   logprob  [n_tokens] of tokens[t]; rank [n_tokens] how many tokens come before
 *            it (a larger logit, or an equal one and a lower index)
 *   entropy  [n_tokens] -sum p log p
 *   top_tokens, top_logprobs  [n_tokens][n_top] the n_top (at most 64) likeliest
 *            tokens in that order, and theirs; -1 and -infinity behind the last
 *            whose logit is above -infinity
 * Any output may be NULL (the top ones with n_top 0), tokens NULL with logprob and
 * rank.  A row with a logit of NaN or +infinity, or with none above -infinity, has no
 * distribution: NaN, rank and top tokens -1.  A token outside [0, vocab): NaN and
 * rank -1.  temperature from 1e-6 to 1e6; at most 2^23 rows of `vocab` (at most 2^24),
 * logits_stride floats apart.  Sums in 64 bits of exponentials in 32.  No output may share memory
 * with an input or another output.  work as for tie_hip_verify_tree. */
size_t tie_hip_token_logprobs_work_bytes(int vocab, int n_tokens, int n_top);
int tie_hip_token_logprobs(const float *logits, size_t logits_stride, int vocab, int n_tokens, const int32_t *tokens,
			   float temperature, int n_top, float *logprob, int32_t *rank, float *entropy, int32_t *top_tokens,
			   float *top_logprobs, void *work, size_t work_bytes, void *stream);

/* Which drafted tokens the target accepts, and the token after them, so that
 * tokens follow the target's distribution whatever the draft proposed.  Token
 * rows first[b] .. first[b + 1] - 1 are a tree: row 0 of a sequence is its root
 * (a token that already stands), parent[t] the node's parent as an index in its
 * sequence (below its own; -1: none, the root), tokens[t] its token.
 *   logits    [n_tokens] rows of `vocab` (the LM head's, for each node)
 *   draft     [n_tokens] rows of `vocab`: the distribution that a node's
 *             children were drawn from, each on its own; NULL: proposed without
 *             probabilities (looked up, or a draft's best)
 *   u_accept, u_sample  F32 [n_tokens] random numbers in [0, 1): for taking the
 *             node, and for the token after it
 * With p = softmax(logits / temperature) of a node and q its draft row, its
 * first max_children children are tried in order: child x is taken when
 * u_accept q(x) M < max(0, p(x) - c q(x)) (c = 0, M = 1 at first); otherwise c
 * += M and M = sum of max(0, p - c q).  Without draft rows: taken when u_accept M
 * < p(x); otherwise x leaves p, and M is what is left.  Where no child is taken, or
 * the path holds max_path nodes, next[b] is the first token whose running sum of
 * the residual (at the path's full length: of p) exceeds u_sample times the
 * whole.  temperature 0: the largest logit (the lowest of equals) alone counts.
 *   path   [n_seqs][max_path] accepted nodes, the root first; -1 behind them
 *   n_keep [n_seqs] how many; next [n_seqs] (0 and -1 for a sequence of no rows)
 * All sums in 64 bits.  No output may share memory with an input.  work as for
 * tie_hip_tree_attention (the same memory will do for both; what is enough for a
 * call is enough for every one of no more tokens and logits). */
size_t tie_hip_verify_tree_work_bytes(int vocab, int n_tokens, int max_children, int with_draft);
int tie_hip_verify_tree(const float *logits, size_t logits_stride, const float *draft, size_t draft_stride, int vocab,
			int n_seqs, int n_tokens, const int32_t *first, const int32_t *tokens, const int32_t *parent,
			const float *u_accept, const float *u_sample, float temperature, int max_children, int max_path,
			int32_t *path, int32_t *n_keep, int32_t *next, void *work, size_t work_bytes, void *stream);

/* ------------------------------------------------------------------ */
/* GGUF models: every MoE layer uploaded once                           */
/* ------------------------------------------------------------------ */

typedef struct tie_hip_model_info {
	char architecture[32]; /* general.architecture */
	int d, F, E, k;        /* embedding_length, expert_feed_forward_length, expert_count, expert_used_count */
	int n_layers;          /* block_count */
	int first_moe_layer;   /* leading_dense_block_count (LFM2), else 0 */
	float norm_eps;        /* attention.layer_norm_rms_epsilon */
	int routing;           /* TIE_HIP_ROUTE_SIGMOID for LFM2, else TIE_HIP_ROUTE_SOFTMAX */
} tie_hip_model_info;

typedef struct tie_hip_model tie_hip_model;

/* Read the MoE shape of a GGUF file (host only, no GPU needed). */
int tie_hip_gguf_inspect(const char *path, tie_hip_model_info *info);

/* One tensor as the library's reader maps it (host only): its GGML type,
 * ne[0..3] (GGUF order, 1 past n_dims), the file offset of its data (the
 * data section starts at the first multiple of general.alignment, default
 * 32, after the tensor infos: gguf_model_map_weights, gguf.c:941-944) and
 * its size in bytes (0 for types the MoE path does not read).  name NULL:
 * only the count.  Returns the file's tensor count, or a negative code. */
int tie_hip_gguf_tensor_info(const char *path, const char *name, int *type, uint64_t ne[4], uint64_t *file_offset,
			     uint64_t *bytes);

/* Map a GGUF file and upload the MoE FFN of every layer from
 * first_moe_layer on: blk.N.ffn_gate_inp / ffn_gate_exps / ffn_up_exps /
 * ffn_down_exps (and exp_probs_b.bias for LFM2) into a tie_hip_layer, and
 * blk.N.ffn_norm.weight to the device, as TIE's model loading maps them
 * (gguf_model_map_weights, gguf.c:892-966; model_load_tensor, model.c:198-235).
 * The file is unmapped before returning. */
int tie_hip_gguf_load(const char *path, tie_hip_model **out);
void tie_hip_model_info_get(const tie_hip_model *m, tie_hip_model_info *info);
/* Layer n's block (NULL for a dense layer) and its device ffn_norm [d] (NULL
 * when the file has none). */
tie_hip_layer *tie_hip_model_layer(tie_hip_model *m, int n);
const float *tie_hip_model_ffn_norm(const tie_hip_model *m, int n);
void tie_hip_model_close(tie_hip_model *m);

/* The largest T that TIE_HIP_PATH_AUTO sends down the exact path (default
 * 14: from 15 tokens on the matrix-core path is the faster one at the 30B shape;
 * 64 or more keeps every decode-sized batch bit-exact). */
int tie_hip_exact_max_tokens(void);
void tie_hip_set_exact_max_tokens(int t);

/* Synchronises `stream` (NULL = the library stream) and reports whether a
 * one-token forward enqueued on it since the last check had a wait between
 * workgroups give up (its outputs NaN): TIE_HIP_EHIP with a message, and
 * the flag cleared; TIE_HIP_OK otherwise.  No counterpart in TIE (its CPU
 * path cannot fail this way). */
int tie_hip_stream_status(void *stream);

/* Debug hook: the next n one-launch one-token forwards wait for a stamp no
 * workgroup writes, with a 64-poll limit, so every wait gives up (and every
 * workgroup still exits): the error path of tie_hip_stream_status. */
void tie_hip_debug_decode_give_up(int n);

/* Debug: force the one-launch one-token kernel's form -- 0 a lane per
 * (row, block) dot, 1 two lanes per dot where the shape's block size and LDS
 * allow them; -1 chosen by the shape (two lanes when every workgroup fits
 * at once).  Both forms give the same bits. */
void tie_hip_debug_decode_form(int form);

/* Debug: the powers of two the layer's matrix-core path scales h and y by
 * (h stored as f16(h 2^-h_shift), y as f16(y 2^-y_shift)), chosen at
 * upload from samples of the gate and down weights. */
int tie_hip_debug_layer_shifts(const tie_hip_layer *layer, int *h_shift, int *y_shift);

/* Make the n-th next allocation fail (n >= 1; 0 disarms): of device memory
 * with TIE_HIP_ENOMEM, of pinned host memory so that the call does without.
 * Host-side fault injection for error-path tests. */
void tie_hip_debug_fail_alloc(int n);

/* Per-kernel timing: while enabled, every kernel of a named section (router,
 * dispatch, expert kernels, combine, ...) is launched with a start and stop
 * event bound to its own dispatch (hipExtLaunchKernel): a section's time is
 * the sum of its kernels' execution times.  Enabling (or disabling) clears
 * what was collected. */
int tie_hip_profile_enable(int on);

/* Sum of event-timed durations and section count per kernel name since the
 * last tie_hip_profile_enable(1); names come back comma-separated in
 * `names`.  Synchronises the device.  Returns the number of names. */
int tie_hip_profile_read(char *names, size_t names_cap, double *total_ms, int *launches, int max_kernels);

/* Host build of the device expf (tie_expf.h) over n inputs, for checking
 * it against the host libm (no GPU needed). */
void tie_hip_host_expf(const float *in, float *out, size_t n);

#ifdef __cplusplus
}
#endif
#endif
