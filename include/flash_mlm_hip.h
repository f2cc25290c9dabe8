/*
 * flash_mlm_hip.h -- C ABI of the MI355X (gfx950) implementation of the
 * flash-mlm fused MLM attention path.
 *
 * Every entry point is `extern "C"`, takes plain device pointers, element
 * counts and strides (in elements, not bytes), launches asynchronously on the
 * HIP stream passed as `void* stream` (NULL = the null stream), allocates no
 * memory, and returns 0 on success, a positive hipError_t on a HIP launch
 * error, or a negative FMLM_E* code when an argument fails the library's own
 * memory-safety checks.  All shape/semantic validation that produces the
 * reference's ValueError messages stays in the host layer above this ABI.
 *
 * Reference interfaces replaced (paths relative to the flash-mlm repository):
 *   fmlm_pack_metadata  <- build_pack_metadata + _build_query_tile_map_from_cu_seqlens
 *                          src/flash_mlm/host/host_utils.py:27-71, 74-107
 *   fmlm_pack           <- _pack_flatten_for_kernel_into / pack_and_pad_main_tensors_for_mlm_compressed
 *                          / pack_for_kernel / pad_packed_main_tensors_for_mlm_compressed
 *                          src/flash_mlm/host/host_utils.py:266-289, 397-420, 423-491, 494-584
 *                          and the dense MLA prefill copy k[:,0].contiguous(),
 *                          src/flash_mlm/host/host.py:206-213
 *   fmlm_unpack         <- unpack_from_kernel, src/flash_mlm/host/host_utils.py:587-615
 *   fmlm_attn_fwd       <- _mlm_compressed_kernel[grid](...) launch, src/flash_mlm/host/host.py:471-521
 *                          and _mlm_main_kernel[grid](...) launch, src/flash_mlm/host/host.py:164-204
 *                          (device bodies src/flash_mlm/mlm_kernel_impl.py:10-62, 65-216, 219-390)
 */
#ifndef FLASH_MLM_HIP_H
#define FLASH_MLM_HIP_H

#include <stdint.h>

#if defined(__GNUC__) || defined(__clang__)
#define FMLM_API __attribute__((visibility("default")))
#else
#define FMLM_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define FMLM_ABI_VERSION 7

/* element types */
enum {
  FMLM_DTYPE_BF16 = 0,
  FMLM_DTYPE_F16 = 1,
  FMLM_DTYPE_F32 = 2
};

/* attention flags (constexpr switches of _mlm_compressed_kernel_impl, mlm_kernel_impl.py:236-238) */
enum {
  FMLM_FLAG_MLA = 1,        /* V is K (one shared latent head for main and context) */
  FMLM_FLAG_PREFILL = 2,    /* skip the cached-context segment */
  FMLM_FLAG_CAUSAL_SEQ = 4, /* sequence b attends to main tokens [0, cu_q[b+1]) */
  FMLM_FLAG_NOSPLIT = 8,    /* key ranges are not split (no records, no merge launch); a
                               schedule is then built with this flag too               */
  FMLM_FLAG_TREE = 32,      /* the call (and its schedule) is for fmlm_attn_tree_fwd         */
  FMLM_FLAG_OWN_RECORDS = 16 /* the schedule has no room for split partial results: every
                               fmlm_attn_fwd on it has this flag too and brings them in
                               its workspace                                           */
};

/* row layouts of a [*, D] tensor addressed by (sequence b, head h, position p) */
enum {
  FMLM_LAYOUT_PADDED = 0, /* row = b*sb + h*sh + p*sn                                  */
  FMLM_LAYOUT_PACKED = 1  /* row = h*sh + (cu_q[b] + p)*sn   (sb ignored)               */
};

/* negative return codes */
enum {
  FMLM_E_ARG = -1,        /* null pointer / negative size / unsupported combination     */
  FMLM_E_DTYPE = -2,      /* unsupported dtype for this entry point                     */
  FMLM_E_HEAD_DIM = -3,   /* unsupported head dimension                                 */
  FMLM_E_ALIGN = -4,      /* pointer or stride not aligned to the element size          */
  FMLM_E_WORKSPACE = -5   /* workspace missing or smaller than fmlm_attn_workspace_bytes */
};

/* ---------------------------------------------------------------------------
 * Library information.
 * ------------------------------------------------------------------------- */
FMLM_API int fmlm_abi_version(void);
/* sizeof(fmlm_attn_params) / sizeof(fmlm_pack_tensor) as compiled, so FFI
 * mirrors can assert their struct layout. */
FMLM_API int fmlm_attn_params_size(void);
FMLM_API int fmlm_pack_tensor_size(void);

/* ---------------------------------------------------------------------------
 * Pack metadata (host_utils.py:27-107).
 *
 * lengths:       [B] int32 (lengths_is_i64 = 0) or int64 (= 1), device.
 * Outputs (device):
 *   lengths_i32   [B]            lengths as int32
 *   aux           [2*B + 6] int32:
 *                   aux[0 .. B]        cu_seqlens  = [0, cumsum(lengths)]
 *                   aux[B+1 .. B+4]    {total_tokens, n_tiles, n_bad_lengths, 0}
 *                   aux[B+5 .. 2B+5]   exclusive tile prefix (internal)
 *   token_indices [B*N] int64    first total_tokens entries = b*N + t, t < L_b, in (b, t) order
 *   batch_ids     [B*ceil(N/block_n)] int32  tile -> sequence, first n_tiles entries valid
 *   tile_starts   [B*ceil(N/block_n)] int32  tile -> packed start cu[b] + j*block_n
 * When any length lies outside [0, N] (n_bad_lengths > 0) only lengths_i32 and
 * aux are written; the caller raises.
 * ------------------------------------------------------------------------- */
FMLM_API int fmlm_pack_metadata(const void* lengths, int32_t lengths_is_i64, int32_t B, int32_t N,
                       int32_t block_n, int32_t* lengths_i32, int32_t* aux,
                       int64_t* token_indices, int32_t* batch_ids, int32_t* tile_starts,
                       void* stream);

/* ---------------------------------------------------------------------------
 * Query tile map from cu_seqlens (host_utils.py:74-107): for every sequence b and
 * j < ceil((cu[b+1]-cu[b]) / block_n), in (b, j) order, batch_ids = b and
 * tile_starts = cu[b] + j*block_n.  At most `capacity` tiles are written;
 * *count (device int32) receives the full tile count.
 * ------------------------------------------------------------------------- */
FMLM_API int fmlm_tile_map(const int32_t* cu_seqlens, int32_t B, int32_t block_n, int32_t capacity,
                           int32_t* batch_ids, int32_t* tile_starts, int32_t* count, void* stream);

/* ---------------------------------------------------------------------------
 * Pack: padded rows (b, h, p < L_b) -> head-major packed rows h*T_pad + cu[b] + p,
 * rows h*T_pad + [T, T_pad) zeroed (host_utils.py:397-420).  Up to 3 tensors
 * per launch (q, k, v).  cu_seqlens == NULL means every sequence has N tokens
 * (then T must equal B*N), which is the dense-prefill copy k[:, 0] -> [B*N, D].
 * Pack and unpack move bytes only: elem_bytes is the element size (1, 2, 4 or 8).
 * ------------------------------------------------------------------------- */
typedef struct fmlm_pack_tensor {
  const void* src; /* source base; element (b, h, p, d) at b*s_sb + h*s_sh + p*s_sn + d */
  int64_t s_sb, s_sh, s_sn;
  void* dst;       /* [heads * T_pad, D] contiguous */
  int32_t heads;   /* heads packed from this tensor (MLA k: 1) */
  int32_t reserved;
} fmlm_pack_tensor;

FMLM_API int fmlm_pack(const fmlm_pack_tensor* tensors, int32_t n_tensors, int32_t elem_bytes, int32_t B,
              int32_t N, int32_t D, const int32_t* cu_seqlens, int32_t T, int32_t T_pad,
              void* stream);

/* ---------------------------------------------------------------------------
 * Unpack: packed rows h*p_sh/D + cu[b] + p -> dst [B, H, N, D] contiguous with
 * zeros where p >= L_b (host_utils.py:587-615).  p_sh = elements between heads
 * of the packed tensor (T*D for [H*T, D]).
 * ------------------------------------------------------------------------- */
FMLM_API int fmlm_unpack(int32_t elem_bytes, const void* packed, int64_t p_sh, void* dst, int32_t B, int32_t H,
                int32_t N, int32_t D, const int32_t* cu_seqlens, void* stream);

/* ---------------------------------------------------------------------------
 * Segment copy, the kernel of a true KV append (InferenceCache.append_kv_cache): for
 * head h < H and segment c < C, rows [src_cu[c], src_cu[c+1]) of src (row h*src_sh/D +
 * i) go to rows [dst_start[c], dst_start[c] + len) of dst (row h*dst_sh/D + i); rows are
 * D elements of elem_bytes.  Offsets are clamped to src_rows / dst_rows rows per head.
 * src == NULL writes zero rows instead (the same segments of dst; src_rows still bounds
 * the offsets src_cu).
 * No counterpart in the reference, which replaces a layer's context on prefill and lists
 * appends with paged KV on its roadmap (README.md:34-41).
 * ------------------------------------------------------------------------- */
FMLM_API int fmlm_copy_segments(int32_t elem_bytes, const void* src, int64_t src_sh, int32_t src_rows,
                                const int32_t* src_cu, void* dst, int64_t dst_sh, int32_t dst_rows,
                                const int32_t* dst_start, int32_t C, int32_t H, int32_t D, void* stream);

/* ---------------------------------------------------------------------------
 * KV append in one launch (InferenceCache.append_kv_cache): for up to 2 tensors (K, V),
 * heads h < H and batches c < C, the merged head-major entry out [H*(t_old+t_new), D]
 * holds, at rows h*(t_old+t_new) + [o_c, o_{c+1}) with o = cu_old + cu_new, the old rows
 * [cu_old[c], cu_old[c+1]) of head h of `old` ([H*t_old, D]) followed by the new rows
 * [cu_new[c], cu_new[c+1]) of head h of `add` ([H*t_new, D]); rows [o_C, t_old+t_new) of
 * every head are zero.  cu_out (C+1 int32, may be NULL) receives o.  Offsets are clamped
 * to the buffers' rows.  No counterpart in the reference, which replaces a layer's
 * context on prefill and lists appends with paged KV on its roadmap (README.md:34-41).
 * ------------------------------------------------------------------------- */
typedef struct fmlm_append_tensor {
  const void* old; /* [H * t_old, D] contiguous */
  const void* add; /* [H * t_new, D] contiguous */
  void* out;       /* [H * (t_old + t_new), D] contiguous */
} fmlm_append_tensor;

FMLM_API int fmlm_kv_append(const fmlm_append_tensor* tensors, int32_t n_tensors, int32_t elem_bytes, int32_t H,
                            int32_t D, int32_t C, int32_t t_old, int32_t t_new, const int32_t* cu_old,
                            const int32_t* cu_new, int32_t* cu_out, void* stream);

/* ---------------------------------------------------------------------------
 * Fused MLM attention forward, dense and packed (mlm_kernel_impl.py:65-216, 219-390).
 *
 * For every sequence b < B, head h < H and query position p < L_b
 * (L_b = cu_seqlens_q[b+1]-cu_seqlens_q[b], or N when cu_seqlens_q == NULL):
 *   keys = [context of b] ++ [main keys of b]
 *   context (skipped with FMLM_FLAG_PREFILL): rows cb*c_sb + h*c_sh + (c0 + j)*c_sn,
 *       j < c1 - c0, where cb = ctx_index[b] clamped to [0, ctx_batch) when ctx_index
 *       is set, else (ctx_batch > 1 ? b : 0), and
 *       (c0, c1) = (cu_seqlens_kv[cb], cu_seqlens_kv[cb+1]) clamped to [0, ctx_rows], or
 *       (0, ctx_len) when cu_seqlens_kv == NULL
 *   main: packed token indices [cu_q[b], cu_q[b+1]), or [0, cu_q[b+1]) with
 *       FMLM_FLAG_CAUSAL_SEQ, addressed through kv_layout
 *   o[b,h,p] = softmax(scale * q[b,h,p] . keys^T) @ values
 * V is K when FMLM_FLAG_MLA is set (v/v_ctx ignored).  bf16/f16 use MFMA with
 * fp32 accumulation and the probabilities rounded to the input type before
 * P.V, as the reference does (mlm_kernel_impl.py:56-58); f32 runs in fp32.
 * L_b is clamped to N (when N > 0) and to total_q - cu_seqlens_q[b].  Rows p >= L_b of
 * the output are not written.
 * ------------------------------------------------------------------------- */
#define FMLM_PAGE_ROWS 64  /* rows per page of a paged context (the kernels' key tile) */

typedef struct fmlm_attn_params {
  int32_t dtype;           /* FMLM_DTYPE_* of q, k, v, contexts and o                */
  int32_t flags;           /* FMLM_FLAG_*                                            */
  int32_t B, H, D;         /* sequences, heads, head dim                             */
  int32_t N;               /* padded per-sequence length                             */
  int32_t total_q;         /* upper bound of sum(L_b) (T or T_pad); B*N when dense   */
  int32_t ctx_len;         /* context length when cu_seqlens_kv == NULL              */
  int32_t ctx_batch;       /* context batch count; 1 => every b uses context batch 0 */
  int32_t ctx_rows;        /* rows per head of a packed context; (c0, c1) are clamped to it */
  int32_t q_layout, o_layout, kv_layout; /* FMLM_LAYOUT_*                          */
  float scale;             /* softmax scale applied to q.k                           */
  const int32_t* cu_seqlens_q;  /* [B+1] or NULL (all sequences have N tokens)      */
  const int32_t* cu_seqlens_kv; /* [ctx_batch+1] or NULL (uniform ctx_len)          */
  const void* q; int64_t q_sb, q_sh, q_sn;
  void* o;       int64_t o_sb, o_sh, o_sn;
  const void* k; int64_t k_sb, k_sh, k_sn;
  const void* v; int64_t v_sb, v_sh, v_sn;
  const void* k_ctx; const void* v_ctx; int64_t c_sb, c_sh, c_sn;
  void* workspace;         /* device scratch for the work schedule                  */
  int64_t workspace_bytes;
  const void* schedule;    /* NULL, or a schedule built by fmlm_attn_schedule for the same
                              cu_seqlens_q contents, B, H, N, total_q, dtype, D, flags,
                              tile_config (with others than it was built for, rows stay
                              unwritten) and kv_layout: then fmlm_attn_fwd launches the attention
                              kernel (plus the split merge) only.  Context lengths may
                              differ; they only steer where key ranges are split.  The
                              buffer also holds split partial results: launches that may
                              overlap need separate schedule buffers.  With
                              FMLM_FLAG_OWN_RECORDS they are in `workspace` instead (at
                              least fmlm_attn_records_bytes, else FMLM_E_WORKSPACE), and
                              launches that overlap only need workspaces of their own */
  const int32_t* ctx_index;  /* [B] context batch of each sequence, or NULL (see above):
                                index-mapped context batching.  No counterpart in the
                                reference, whose roadmap lists it ("variable context
                                batch sizes", README.md:34-36)                         */
  /* Paged context (NULL block table: contiguous context as above).  Context batch cb has
   * cu_seqlens_kv[cb+1] - cu_seqlens_kv[cb] rows (or ctx_len); its row j lives in page
   * ctx_block_table[cb * ctx_pages_per_batch + j / FMLM_PAGE_ROWS], row j % FMLM_PAGE_ROWS:
   * element page * ctx_page_stride + h * c_sh + (j % FMLM_PAGE_ROWS) * c_sn of k_ctx /
   * v_ctx.  ctx_rows is then the number of pages in the pool (page ids are clamped to it).
   * bf16/f16 with linear main keys only.  No counterpart in the reference, whose roadmap
   * lists paged KV (README.md:41).                                                     */
  const int32_t* ctx_block_table;
  int64_t ctx_page_stride;
  int32_t ctx_pages_per_batch;
  /* Tile configuration of the bf16/f16 attention kernel: 0 = chosen by the library from
   * the head dim and the query rows (D = 64 and 128: configuration 3 when total_q <=
   * 64 * B, i.e. sequences of at most 64 query rows on average, or when the 128-row
   * workgroups of a dense call would fill at most half of the GPU, else 1; D = 256: 2 when
   * 64-row workgroups would be more than 256 and total_q > 64 * B, else 1; other head dims: 1); k >= 1
   * forces compiled configuration k of the head dim (fmlm_attn_workspace_bytes returns
   * FMLM_E_ARG for a k that does not exist).  Configurations, as (query rows per
   * workgroup, waves per workgroup): D = 16, 32: 1 = (128, 4); D = 64: 1 = (128, 4),
   * 2 = (256, 8), 3 = (64, 4), 4 = (256, 8) ping-pong; D = 128: 1 = (128, 4),
   * 2 = (256, 8), 3 = (64, 4), 4 = (128, 8), 5 = (256, 8) ping-pong; D = 256:
   * 1 = (64, 4), 2 = (128, 8); MLA D = 512: 1 = (128, 8), in packed calls of at most 4096
   * (head, position) rows (64, 8).  Tree calls (FMLM_FLAG_TREE): 1 = (64, 4), which 0 is, D = 256 also
   * 2 = (128, 8): fmlm_attn_tree_tile says when it pays.
   * Ping-pong: the 8 waves run as
   * two groups half a key tile apart, so that one wave of each SIMD computes softmax
   * while the other issues MFMAs.  Replaces the reference's autotuned
   * BLOCK_M / BLOCK_N / num_warps (mlm_kernel.py:57-166).  Ignored by f32 inputs.       */
  int32_t tile_config;
  /* Row statistics for the backward: NULL, or H * total_q floats that fmlm_attn_fwd fills
   * with each real query row's log2-sum-exp, row p of sequence b and head h at
   * h * total_q + q0_b + p (q0_b = cu_seqlens_q[b], or b * N without cu_seqlens_q):
   * log2(sum over its keys of 2^z), z = scale * log2(e) * q.k as the forward kernel
   * computes it (fp32 accumulation); +inf for a row without keys.
   * fmlm_attn_bwd given the same block reads it instead of recomputing it.  No
   * counterpart in the reference, whose kernels return o only.                        */
  float* lse;
} fmlm_attn_params;

/* Bytes of device workspace (and of a schedule buffer) fmlm_attn_fwd needs for these
 * parameters (>= 0), or < 0 on unsupported dtype / head dim.  A dense call
 * (cu_seqlens_q == NULL) also runs without: its key ranges are then not split. */
FMLM_API int64_t fmlm_attn_workspace_bytes(const fmlm_attn_params* p);

/* The part of fmlm_attn_workspace_bytes that holds split partial results, or < 0 as above.
 * 0 when the call cannot split: with FMLM_FLAG_NOSPLIT set it then does the same with one
 * launch less, in a smaller schedule and workspace (for a packed call by its own context
 * sizes: without the flag it must still run a schedule built for longer contexts). */
FMLM_API int64_t fmlm_attn_records_bytes(const fmlm_attn_params* p);

/* Build the work schedule (one entry per query tile of the kernel's own tile size over
 * the real rows of every sequence) into `schedule` (fmlm_attn_workspace_bytes bytes, with
 * FMLM_FLAG_OWN_RECORDS less fmlm_attn_records_bytes; FMLM_E_WORKSPACE when it is smaller)
 * so later fmlm_attn_fwd calls with p->schedule = schedule skip rebuilding it.  No counterpart in the reference (its tile map is PackMetadata.batch_ids_q /
 * q_tile_starts_q at block_n granularity, host_utils.py:74-107). */
FMLM_API int fmlm_attn_schedule(const fmlm_attn_params* p, void* schedule, int64_t schedule_bytes,
                                void* stream);

FMLM_API int fmlm_attn_fwd(const fmlm_attn_params* p, void* stream);

/* ---------------------------------------------------------------------------
 * fmlm_attn_fwd without a workspace, for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid allocation).
 * No counterpart in the reference.  Same parameters and results as fmlm_attn_fwd;
 * p->workspace and p->schedule are ignored.  The work schedule and the split-KV partial
 * results live in a device array owned by the library, FMLM_NOALLOC_SCRATCH_BYTES per
 * GPU, held until the process ends; the schedule is rebuilt on every call.  When the
 * split records would not fit, fewer key ranges are split (or none); a call whose
 * unsplit schedule does not fit returns FMLM_E_WORKSPACE.  Every packed call on a GPU
 * shares that GPU's array: calls that may overlap on one GPU (different streams, or host
 * threads) race and must be serialised by the caller.  Dense calls (cu_seqlens_q == NULL)
 * do not split and do not use the array: they may overlap any other.  Allocates nothing.
 * ------------------------------------------------------------------------- */
#define FMLM_NOALLOC_SCRATCH_BYTES (16 << 20)

FMLM_API int fmlm_attn_fwd_noalloc(const fmlm_attn_params* p, void* stream);

/* ---------------------------------------------------------------------------
 * Attention backward.  No counterpart in the reference, whose roadmap lists
 * backpropagation (README.md:26-28); it differentiates fmlm_attn_fwd for the same
 * parameter block p (p->o holding that call's output):
 *   dq      rows laid out like q (q_layout) with the dq strides: every real row
 *   dk, dv  main-key rows laid out like k / v (kv_layout) with the dk / dv strides: every
 *           key row some query attends to.  With FMLM_FLAG_MLA dk receives the gradient
 *           of K and of V (V is K) and dv is unused.  Keys with head stride 0 (the MLA
 *           latent) are shared by all heads, and so is their gradient row (dk_sh = 0).
 *   dk_ctx, dv_ctx  the context's gradient, laid out like k_ctx / v_ctx (c_sb, c_sh,
 *           c_sn), or NULL to skip it: rows [c0, c1) of every context batch.  With a
 *           paged context (ctx_block_table) they are float32 buffers laid out like the
 *           pool, zeroed by the caller, that the kernel adds into atomically: a page used
 *           by several context batches receives the sum of their gradients.
 * Rows not listed are not written.  dout is laid out like o (o_layout).
 * bf16 / f16 / f32, D in {16, 32, 64, 128, 256, 512}: MFMA kernels, except 16-bit D = 16,
 * D = 512 (16-bit without MLA, f32) and f32 with a paged context (which fmlm_attn_fwd does
 * not run), which take SIMT kernels; with FMLM_FLAG_CAUSAL_SEQ the main keys must be packed
 * (kv_layout PACKED).
 * workspace: fmlm_attn_bwd_workspace_bytes(p) bytes (per-row softmax statistics, the
 *           tile tables of the two kernels and a 64-byte record per tile).
 * ------------------------------------------------------------------------- */
typedef struct fmlm_attn_grads {
  const void* dout; int64_t do_sb, do_sh, do_sn;
  void* dq;  int64_t dq_sb, dq_sh, dq_sn;
  void* dk;  int64_t dk_sb, dk_sh, dk_sn;
  void* dv;  int64_t dv_sb, dv_sh, dv_sn;
  void* dk_ctx;
  void* dv_ctx;
  void* workspace;
  int64_t workspace_bytes;
} fmlm_attn_grads;

FMLM_API int fmlm_attn_grads_size(void);  /* sizeof(fmlm_attn_grads), for bindings */
FMLM_API int64_t fmlm_attn_bwd_workspace_bytes(const fmlm_attn_params* p);
FMLM_API int fmlm_attn_bwd(const fmlm_attn_params* p, const fmlm_attn_grads* g, void* stream);
/* The same for gradients that were not zeroed: the rows that fmlm_attn_bwd does not write
 * become zero too, namely the padding rows [L_b, N) of padded q / k / v gradients, the rows
 * of packed ones (and of a packed context's) before the first and after the last sequence
 * (context batch).  Rows per head of a packed gradient: its head stride / row stride.
 * Gradients of keys shared by all heads (head stride 0) and of paged contexts still have to
 * be zeroed by the caller. */
FMLM_API int fmlm_attn_bwd_fill(const fmlm_attn_params* p, const fmlm_attn_grads* g, void* stream);

/* ---------------------------------------------------------------------------
 * Norms of queries and keys for each head with the position rotation (no counterpart in
 * the reference, whose entry points take q and k as they are).  A row is the D elements x
 * of one head and token; in fp32, rounded once to dtype:
 *   n_d = x_d (mean(x^2) + eps)^-1/2 w_d            (FMLM_NR_NORM; else n = x)
 *   pairs (a, b) of n's first rotary_dim elements -> (a c - b s, a s + b c),
 *   c, s = cos / sin[angle row, i]; pair i is elements (i, i + rotary_dim / 2), or
 *   (2i, 2i + 1) with FMLM_NR_INTERLEAVED.
 * Rows.  PADDED: row b * N + p at b * sb + h * sh + p * sn; rows p >= L_b (cu_seqlens) are
 * written as zeros.  PACKED: token t at h * sh + t * sn, which is token token_indices[t] =
 * b * N + p of the padded batch (NULL: B = 1 and t = p).
 * Angle row of a token: positions[i] (i: the packed token, or b * N + p without
 * cu_seqlens), else offsets[b] + p, else p; clamped to [0, table_rows).
 * D in {16, 32, 64, 128, 256, 512}; rotary_dim a multiple of 16; rows, cos and sin 16-byte
 * aligned with unit stride along D.
 * ------------------------------------------------------------------------- */
enum {
  FMLM_NR_NORM = 1,
  FMLM_NR_INTERLEAVED = 2,
  FMLM_NR_POSITIONS_I64 = 4, /* positions are int64 (else int32) */
  FMLM_NR_OFFSETS_I64 = 8    /* offsets are int64 (else int32)   */
};

typedef struct fmlm_norm_rope_tensor {
  const void* x;  int64_t x_sb, x_sh, x_sn;
  void* y;        int64_t y_sb, y_sh, y_sn;    /* forward: the rows out; backward: dx */
  const void* dy; int64_t dy_sb, dy_sh, dy_sn; /* backward only: the gradient of the rows out */
  const void* weight; /* gains, or NULL for 1: [D] (w_sh = 0) or [heads, D] (w_sh = D) */
  void* dweight;      /* backward: laid out like weight, or NULL to skip it */
  int64_t w_sh;
  int32_t heads;      /* 0: no such tensor */
  int32_t reserved;
} fmlm_norm_rope_tensor;

typedef struct fmlm_norm_rope_params {
  int32_t dtype;   /* FMLM_DTYPE_* of the rows        */
  int32_t w_dtype; /* FMLM_DTYPE_* of gains and dweight */
  int32_t flags;   /* FMLM_NR_*                       */
  int32_t layout;  /* FMLM_LAYOUT_*                   */
  int32_t B, N, D;
  int32_t rotary_dim; /* 0: no rotation */
  int64_t rows;       /* B * N, or packed tokens      */
  int64_t table_rows;
  float eps;
  int32_t n_positions; /* entries of positions: a padded row past them is no token; 0: not said */
  const float* cos; /* [table_rows, rotary_dim / 2] fp32 */
  const float* sin;
  const int32_t* cu_seqlens;    /* [B+1] or NULL */
  const int64_t* token_indices; /* see above, or NULL */
  const void* positions;        /* or NULL */
  const void* offsets;          /* [B], or NULL */
  fmlm_norm_rope_tensor q, k;
  void* workspace; /* backward: fmlm_norm_rope_bwd_workspace_bytes(p) bytes (partial sums of dw) */
  int64_t workspace_bytes;
} fmlm_norm_rope_params;

FMLM_API int fmlm_norm_rope_params_size(void);
FMLM_API int fmlm_norm_rope(const fmlm_norm_rope_params* p, void* stream);
/* Gradients of the same call: x and dy in, dx to y, dweight where given; dx of padding rows
 * is zero.  Sums are taken in one order: the same call gives the same bits. */
FMLM_API int64_t fmlm_norm_rope_bwd_workspace_bytes(const fmlm_norm_rope_params* p);
FMLM_API int fmlm_norm_rope_bwd(const fmlm_norm_rope_params* p, void* stream);

/* ---------------------------------------------------------------------------
 * Block table and slots of a step's new tokens (no counterpart in the reference, whose
 * roadmap lists paged KV, README.md:41).  Request b has old_lens[b] tokens in its context
 * pages (FMLM_PAGE_ROWS rows each) and gets L_b = cu_seqlens[b+1] - cu_seqlens[b] new ones,
 * or those of them with keep[t] != 0.  Requests take the pages they lack from free_pages
 * in order:
 *   have_b = ceil(old_b / 64), need_b = ceil((old_b + new_b) / 64) - have_b
 *   block_table[b, i] = table_in[b, i] for i < have_b, then free_pages[sum of the needs
 *       before b + i - have_b], and -1 from i = have_b + need_b on
 *   slot_mapping[t] = page * 64 + row of the token's place (old_b + its rank among the kept
 *       tokens of b), -1 for a token that is not kept
 *   positions[t] = old_b + p, new_lens[b] = old_b + new_b, cu_kv its prefix sums
 * table_in == NULL: no request has pages yet (old_lens must be 0).  A request that does not
 * fit its table row or finds no free page keeps the tokens that fit (the others' slots are
 * -1).  summary: {pages taken, pages lacking in free_pages, requests with an old length
 * out of range or more tokens than the row holds, tokens stored}.
 * workspace: fmlm_block_table_workspace_bytes(p) bytes.
 * ------------------------------------------------------------------------- */
enum {
  FMLM_BT_OLD_I64 = 1,   /* old_lens are int64 (else int32)   */
  FMLM_BT_TABLE_I64 = 2, /* table_in is int64 (else int32)    */
  FMLM_BT_FREE_I64 = 4   /* free_pages are int64 (else int32) */
};

typedef struct fmlm_block_table_params {
  int32_t flags;
  int32_t B, N;      /* requests, padded length of their new tokens */
  int32_t T;         /* new tokens: cu_seqlens[B] */
  int32_t max_pages; /* entries of a row of block_table */
  int32_t in_pages;  /* entries of a row of table_in */
  int32_t n_free;
  int32_t reserved;
  const void* old_lens;         /* [B] */
  const int32_t* cu_seqlens;    /* [B+1] */
  const int64_t* token_indices; /* [T] b * N + p (fmlm_pack_metadata) */
  const uint8_t* keep;          /* [T] or NULL */
  const void* table_in;         /* [B, in_pages] or NULL */
  const void* free_pages;       /* [n_free] */
  int32_t* block_table;         /* [B, max_pages] */
  int64_t* slot_mapping;        /* [T] */
  int32_t* positions;           /* [T] */
  int32_t* new_lens;            /* [B] */
  int32_t* cu_kv;               /* [B+1] */
  int32_t* summary;             /* [4] */
  void* workspace;
  int64_t workspace_bytes;
} fmlm_block_table_params;

FMLM_API int fmlm_block_table_params_size(void);
FMLM_API int64_t fmlm_block_table_workspace_bytes(const fmlm_block_table_params* p);
FMLM_API int fmlm_block_table(const fmlm_block_table_params* p, void* stream);

/* ---------------------------------------------------------------------------
 * Paged append: for up to 2 tensors (K, V), head h and token t < T, the D elements (h, t) of
 * src go to row slots[t] of head h of the pool [heads, pool_rows, D]; slots outside [0,
 * pool_rows) are skipped.  src rows: PADDED b * sb + h * sh + p * sn for token_indices[t] =
 * b * N + p, PACKED h * sh + t * sn.  Moves bytes only.
 * ------------------------------------------------------------------------- */
typedef struct fmlm_paged_tensor {
  const void* src;
  int64_t s_sb, s_sh, s_sn;
  void* pool;
  int64_t batch; /* PADDED: sequences in src, to which those of token_indices are clamped; 0: not said */
} fmlm_paged_tensor;

FMLM_API int fmlm_paged_append(const fmlm_paged_tensor* tensors, int32_t n_tensors, int32_t elem_bytes, int32_t heads,
                               int32_t D, int32_t T, int32_t N, int32_t layout, const int64_t* token_indices,
                               const int64_t* slots, int64_t pool_rows, void* stream);

/* ---------------------------------------------------------------------------
 * Trees of drafted tokens.  parents[t] (int32 or int64) is the index, within its sequence,
 * of the token that token t follows, -1 for a root.  A parent has to come before its child:
 * other values count in *n_bad (may be NULL) and are taken as -1.
 *   mask[t * words + j / 64], bit j % 64: token j of t's sequence is t or an ancestor of it
 *   positions[t] = (ctx_lens ? ctx_lens[b] : 0) + number of t's ancestors
 * words >= ceil(N / 64); at most FMLM_MAX_TREE tokens in a sequence (N).
 * ------------------------------------------------------------------------- */
#define FMLM_MAX_TREE 256

FMLM_API int fmlm_tree_mask(const void* parents, int32_t parents_i64, const int32_t* cu_seqlens, int32_t B, int32_t N,
                            int32_t T, int32_t words, const void* ctx_lens, int32_t ctx_lens_i64, uint64_t* mask,
                            int32_t* positions, int32_t* n_bad, void* stream);

/* Attention of drafted trees: fmlm_attn_fwd's packed call p (linear main keys, no
 * FMLM_FLAG_PREFILL or CAUSAL_SEQ) with FMLM_FLAG_TREE, in which token i of a sequence attends
 * to [its context || the main tokens j of its sequence with mask bit j set]; bits at or past
 * the sequence's end are ignored.  A row that sees no key has output 0.  At most FMLM_MAX_TREE
 * tokens in a sequence (N, or total_q where N is 0).  p->lse is not used; no backward.
 * Up to D = 256 the attention kernel masks the main keys itself.  For D = 512 (MLA) a second
 * kernel computes the tree's part, and the context's part goes through tree_workspace:
 * fmlm_attn_tree_workspace_bytes(p) bytes (0 in the first case). */
FMLM_API int fmlm_attn_tree_tile(const fmlm_attn_params* p); /* the tile_config that the call's
                               shape and context ask for (p's own when set; 0: there is no
                               choice), or FMLM_E_ARG.  Set it before the sizes are asked for */
FMLM_API int64_t fmlm_attn_tree_workspace_bytes(const fmlm_attn_params* p);
FMLM_API int fmlm_attn_tree_fwd(const fmlm_attn_params* p, const uint64_t* mask, int32_t words, void* tree_workspace,
                                int64_t tree_workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Window attention.  fmlm_attn_fwd's call p with a limit on what a query sees: keys are numbered
 * from the first context row on, the main keys after them, and the query of token i of a
 * sequence with n context rows is at position n + i (FMLM_WINDOW_APPENDED: n - L + i, the
 * sequence's L tokens are its last context rows already and there are no main keys).  The
 * query at position s sees key j if
 *   j <= s + right  and  (j >= s - left  or  j < sinks).
 * left, right < 0: no limit.  A row that sees no key has output 0.
 *
 * p: bf16 or fp16, D = 32, 64, 128 or 256, a finite scale, flags 0, packed sequences (cu_seqlens_q); q, k and v
 * padded or packed, the output packed or padded; main keys linear; the context packed
 * (cu_seqlens_kv), paged, or none (cu_seqlens_kv NULL, ctx_len 0); ctx_index as there.  p->schedule
 * and tile_config are not used.
 *
 * 4-bit context (FMLM_WINDOW_FP4, paged only): rows of E2M1 codes, element 2i in the low and
 * 2i + 1 in the high half of byte i, and for every 32 elements of a row the scale 2^(x - 127) as a
 * byte x.  p->k_ctx / v_ctx are the codes, c_sh, c_sn and ctx_page_stride count elements (so
 * offset / 2 bytes of codes, offset / 32 scales).  fp16 holds every value of scale bytes 104 to
 * 140, bf16 of those up to 252.
 * ------------------------------------------------------------------------- */
enum { FMLM_WINDOW_APPENDED = 1, FMLM_WINDOW_FP4 = 2 };

typedef struct fmlm_window {
  int32_t left, right, sinks, flags;
  const uint8_t* k_scales; /* FMLM_WINDOW_FP4 */
  const uint8_t* v_scales;
  void* o_low; /* NULL, or laid out like o: what o's rounding took away (o + o_low is the result to
                  twice the type's digits).  A backward with it has delta = rowsum(do o) without
                  that rounding, whose part in dq and dk is largest in narrow windows */
} fmlm_window;

FMLM_API int fmlm_window_size(void);
/* p->workspace: fmlm_window_workspace_bytes(p, w) (0 where key ranges are not split; p->lse, and
 * FMLM_FLAG_NOSPLIT in p->flags, rule that out) */
FMLM_API int64_t fmlm_window_workspace_bytes(const fmlm_attn_params* p, const fmlm_window* w);
FMLM_API int fmlm_window_fwd(const fmlm_attn_params* p, const fmlm_window* w, void* stream);
/* Gradients of a call without a context whose forward stored p->lse; g as in fmlm_attn_bwd (no
 * dk_ctx, dv_ctx), of which it writes every row of every sequence, padding rows as zeros.
 * g->workspace: H * total_q floats. */
FMLM_API int fmlm_window_bwd(const fmlm_attn_params* p, const fmlm_window* w, const fmlm_attn_grads* g, void* stream);

/* ---------------------------------------------------------------------------
 * Appends to a paged context with the position rotation on the way: of the packed tokens t, with
 * c, s = cos, sin[positions[t]] (rows of rotary_dim / 2 floats), the first rotary_dim elements of
 * q's and k's rows become (a c - b s, a s + b c) for the pairs (a, b) = (i, i + rotary_dim / 2), or
 * (2i, 2i + 1) with FMLM_AP_INTERLEAVED.  q goes to q.dst (padding rows as zeros), k and v to row
 * slots[t] of their pools (heads pool_rows rows apart); slots outside [0, pool_rows) are not
 * stored.  Positions are clamped to the table_rows of the tables.  With FMLM_AP_FP4 the pools hold
 * 4-bit rows (see above): the scale of a block is the smallest 2^e with which its magnitudes are
 * below 7 2^e, e within [-23, 13] (fp16) or [-125, 125] (bf16); codes are rounded to nearest
 * even, to at most 6; infinities count as the type's largest value, NaN as 0.
 * k's values are rotated in 64 bits there, so that no rounding but the codes' decides a code.
 * A tensor with dst NULL is left out; cos NULL (rotary_dim 0): nothing is rotated.
 * ------------------------------------------------------------------------- */
enum { FMLM_AP_INTERLEAVED = 1, FMLM_AP_FP4 = 2, FMLM_AP_POSITIONS_I64 = 4 };

typedef struct fmlm_append_rows {
  const void* src;
  int64_t s_sb, s_sh, s_sn; /* padded: b*sb + h*sh + p*sn, packed: h*sh + t*sn                */
  void* dst;                /* q: rows of its own strides; k, v: the pool                    */
  int64_t d_sb, d_sh, d_sn; /* q only                                                        */
  uint8_t* scales;          /* k, v with FMLM_AP_FP4                                         */
} fmlm_append_rows;

typedef struct fmlm_append_params {
  int32_t dtype, flags, layout;
  int32_t B, H, N, D, rotary_dim, T;
  int32_t reserved;
  int64_t table_rows, pool_rows;
  const float* cos;
  const float* sin;
  const void* positions;      /* [T]                                                         */
  const int32_t* cu_seqlens;  /* [B + 1]                                                     */
  const int64_t* slots;       /* [T]                                                         */
  fmlm_append_rows q, k, v;
} fmlm_append_params;

FMLM_API int fmlm_append_params_size(void);
FMLM_API int fmlm_rotate_append(const fmlm_append_params* p, void* stream);

/* The values of `rows` 4-bit rows of D elements (contiguous codes and scales) of one or two tensors,
 * as bf16 or fp16. */
typedef struct fmlm_fp4_rows {
  const uint8_t* codes;
  const uint8_t* scales;
  void* out;
} fmlm_fp4_rows;

FMLM_API int fmlm_fp4_values(int32_t dtype, const fmlm_fp4_rows* tensors, int32_t n_tensors, int64_t rows, int32_t D,
                             void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FLASH_MLM_HIP_H */
