/*
 * dsalt_b200: B200 (sm_100a) kernels for the DSALT sparse-attention forward.
 *
 * C ABI: plain pointers, sizes and a CUDA stream (passed as void*). All pointers are
 * device pointers unless stated otherwise; nothing here allocates device memory —
 * callers pass output buffers and a workspace sized by the *_workspace_bytes queries.
 * Every entry point returns DSALT_OK (0) or an error code and leaves a message for
 * dsalt_last_error(). Kernels are launched asynchronously on `stream`.
 *
 * Each function cites the reference (LeonardoCofone/dsalt) interface it replaces.
 */
#ifndef DSALT_B200_H
#define DSALT_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define DSALT_F32 0
#define DSALT_BF16 1
#define DSALT_F16 2

/* status codes */
#define DSALT_OK 0
#define DSALT_ERR_INVALID 1       /* bad shape, dtype, stride, alignment or pointer */
#define DSALT_ERR_UNSUPPORTED 2   /* valid request outside what the kernels implement */
#define DSALT_ERR_CUDA 3          /* a CUDA runtime/driver call failed */
#define DSALT_ERR_WORKSPACE 4     /* workspace smaller than the *_workspace_bytes query */
#define DSALT_ERR_DEVICE 5        /* a kernel gave up a bounded wait (see dsalt_device_status) */

/* selection modes */
#define DSALT_SELECT_GLOBAL 0       /* one landmark set per (head, sequence) */
#define DSALT_SELECT_BLOCK_CAUSAL 1 /* one landmark set per (head, block of queries) */

/* norm rounding of the selection signals */
#define DSALT_NORM_F32 0   /* fp32 norms (CUDA autocast runs `norm` in fp32) */
#define DSALT_NORM_INPUT 1 /* norms rounded to the input dtype (bf16/fp16 `norm` outside autocast) */

const char* dsalt_last_error(void);
int dsalt_version(void);

/* Reads (and clears, when `clear` != 0) the device status word that kernels set when a
 * bounded wait gives up. Synchronises `stream`. 0 = no error. The device addresses of this
 * word and of the no-allocation scratch array are looked up once per device and kept for
 * the life of the process: do not use the library across a cudaDeviceReset. */
int dsalt_device_status(int* status_out, int clear, void* stream);
/* Queues a copy of the device status word into host memory `status_host` (page-locked, so
 * that the copy is asynchronous) on `stream` and returns without synchronising; the value
 * is there once the stream has passed this point (e.g. an event recorded after the call
 * has completed). Lets a caller check every step without stalling the stream. */
int dsalt_device_status_async(int* status_host, void* stream);

/*
 * Window widths and selection signals, one pass over x and v.
 * Replaces DSALTAttention._window_sizes(x, floor=True)
 *   (dsalt/modules/dsalt_attention.py:270-284, win_gate at :223)
 * and the norms of hybrid_scores_per_head / _token_signals
 *   (dsalt/kernels/landmark_tokens_ker.py:47,52; results/causal_landmark_check.py:68-79).
 *
 * x        [T, d_model] (row stride x_stride elements), dtype x_dtype
 * gate_w   [d_model], gate_b [1]: win_gate weight/bias in gate_dtype; the logit is
 *          computed in gate_dtype (x converted to gate_dtype first, as autocast does)
 * v        [T, n_kv*head_dim] value projection x·W_Vᵀ (row stride v_stride), dtype v_dtype
 * w_out    [T] int32 widths, xnorm_out [T] fp32, vnorm_out [T, n_kv] fp32
 * logit_out [T] fp32 (nullable): the rounded win_gate logit
 * logit_in  [T] in gate_dtype (nullable): the win_gate logit as the caller computed it
 *          (e.g. torch's `win_gate(x)` under autocast, the reference's own op); the widths
 *          are then computed from it (gate_w / gate_b are still passed but no longer
 *          affect any output). Without it the logit is the float64-accumulated dot
 *          product rounded once to gate_dtype, which a library GEMV that accumulates in
 *          fp32 can round to the neighbouring value.
 */
int dsalt_token_signals(const void* x, int x_dtype, int64_t T, int d_model, int64_t x_stride,
                        const void* gate_w, const void* gate_b, int gate_dtype, int n_min, int n_max,
                        const void* v, int v_dtype, int64_t v_stride, int n_kv, int head_dim, int norm_mode,
                        int32_t* w_out, float* xnorm_out, float* vnorm_out, float* logit_out,
                        const void* logit_in, void* stream);

/*
 * Landmark selection.
 * DSALT_SELECT_GLOBAL replaces _compute_landmark_indices
 *   (dsalt/kernels/selectors.py:75-134) with hybrid_scores_per_head
 *   (dsalt/kernels/landmark_tokens_ker.py:19-61): statistics over all T packed tokens,
 *   top-k per (head, sequence) among tokens with seq_off >= w.
 * DSALT_SELECT_BLOCK_CAUSAL replaces the per-block _select of
 *   results/causal_landmark_check.py:82-113 (driven at :176-186): block b of each
 *   sequence draws from positions [0, b*block) with that prefix's statistics.
 *
 * xnorm [T], vnorm [T, n_kv], w [T] (int32), alpha [n_heads] (sigmoid(alpha_w), fp32)
 * cu_seqlens [n_seqs+1] int32 (device), max_seqlen: host upper bound of sequence lengths
 * lmk_out [n_heads, n_sets, k] int32: positions within the sequence, ascending, -1 padded.
 *   n_sets = n_seqs (global) or sum over sequences of ceil(L/block) (block-causal,
 *   numbered sequence after sequence).
 * zx_out [T], zv_out [T, n_kv] (nullable, global mode only): the standardized signals.
 * Tie rule: equal scores are taken lowest position first.
 */
size_t dsalt_select_workspace_bytes(int mode, int64_t T, int n_seqs, int max_seqlen, int n_heads, int n_kv,
                                    int k, int block);
int dsalt_select_landmarks(int mode, const float* xnorm, const float* vnorm, const int32_t* w,
                           const float* alpha, const int32_t* cu_seqlens, int n_seqs, int64_t T, int max_seqlen,
                           int n_heads, int n_kv, int k, int block, int32_t* lmk_out, float* zx_out,
                           float* zv_out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Sparse attention forward over A(i) = W(i) ∪ L(i).
 * Replaces dsalt_triton_attention / DSALTAttentionFunction.forward
 *   (dsalt/kernels/dsalt_triton_attn.py:259-311, :337-349) and _dsalt_fwd_kernel (:27-169),
 *   including _build_landmark_kv (dsalt/kernels/selectors.py:137-159) and
 *   _build_seq_block_map (selectors.py:37-67), which are done inside.
 *
 * q [T, n_heads, head_dim], k/v [T, n_kv, head_dim] (token strides q_stride, kv_stride in
 *   elements; heads contiguous), dtype DSALT_BF16 / DSALT_F16 (tensor cores; head_dim 64 or
 *   128) or DSALT_F32 (fp32 CUDA cores; head_dim 32, 64, 128 or 256). GQA: head h uses kv
 *   head h / (n_heads / n_kv).
 * w [T] int32 window widths (clamped to >= 1 inside).
 * lmk [n_heads, n_sets, k_lmk] int32 positions within the sequence, -1 = none. For the
 *   bf16/fp16 path every set must list its positions ascending with the -1 entries last
 *   (the format dsalt_select_landmarks writes); the fp32 path accepts any order.
 *   lmk_block = 0: one set per sequence; > 0: one set per lmk_block queries.
 * lmk_bias [n_heads, n_sets, k_lmk] fp32 (nullable): added to landmark logits.
 * out [T, n_heads, head_dim] in out_dtype; lse [T, n_heads] fp32 (nullable).
 */
size_t dsalt_attention_workspace_bytes(int64_t T, int n_seqs, int n_heads, int k_lmk, int lmk_block);
int dsalt_attention_fwd(const void* q, const void* k, const void* v, int dtype, int64_t T, int n_heads, int n_kv,
                        int head_dim, int64_t q_stride, int64_t kv_stride, const int32_t* w, const int32_t* lmk,
                        const float* lmk_bias, int k_lmk, int lmk_block, const int32_t* cu_seqlens, int n_seqs,
                        int max_seqlen, void* out, int out_dtype, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream);

/*
 * Backward of the sparse attention forward above.
 * Replaces dsalt_triton_backward / DSALTAttentionFunction.backward
 *   (dsalt/kernels/dsalt_triton_bwd.py:219-323, dsalt_triton_attn.py:313-327), i.e.
 *   _dsalt_bwd_preprocess (:18-49) and _dsalt_bwd_kernel (:52-216).
 *
 * q, k, v, w, lmk, lmk_bias, lmk_block, cu_seqlens as for the forward (lmk in the forward's
 *   ascending format); n_sets = lmk's second extent. out [T, n_heads, head_dim] is the
 *   forward's output in out_dtype and dout [T, n_heads, head_dim] its gradient in
 *   dout_dtype (both contiguous); lse [T, n_heads] fp32 the forward's log-sum-exp (natural
 *   log, -inf for rows with no key). Outputs (fp32, overwritten): dq [T, n_heads, head_dim],
 *   dk / dv [T, n_kv, head_dim] (summed over the heads of each kv group), d_bias
 *   [n_heads, n_sets, k_lmk] (nullable). head_dim 64 or 128; lmk_block a multiple of 64.
 *   S = q·kᵀ and dO·vᵀ on the tensor cores (mma.sync, fp32 accumulate) when q/k/v and dout
 *   share a 16-bit dtype, on CUDA cores otherwise; the gradient products on CUDA cores in
 *   fp32; dk, dv and d_bias accumulate with atomic adds, so their last bits vary from run to
 *   run.
 */
size_t dsalt_attention_bwd_workspace_bytes(int64_t T, int n_seqs);
int dsalt_attention_bwd(const void* q, const void* k, const void* v, int dtype, int64_t T, int n_heads, int n_kv,
                        int head_dim, int64_t q_stride, int64_t kv_stride, const void* out, int out_dtype,
                        const void* dout, int dout_dtype, const float* lse, const int32_t* w, const int32_t* lmk,
                        const float* lmk_bias, int k_lmk, int lmk_block, int n_sets, const int32_t* cu_seqlens,
                        int n_seqs, float* dq, float* dk, float* dv, float* d_bias, void* workspace,
                        size_t workspace_bytes, void* stream);

/*
 * Training-time sparse attention with differentiable selectors (forward and backward).
 * Replaces dsalt_triton_train_attention / DSALTTrainAttentionFunction
 *   (dsalt/kernels/dsalt_triton_train.py:583-782): _train_fwd_kernel (:74-217),
 *   _train_bwd_preprocess, _train_bwd_kernel and _train_bwd_dkdv_kernel (:220-490).
 *
 * q [T, n_heads, head_dim], k/v [T, n_kv, head_dim] as for the forward above (any of bf16,
 *   fp16, fp32; head_dim 64 or 128). The forward runs bf16 / fp16 inputs with
 *   0 <= win_edge <= 4 on the tensor cores (P rounded to the input dtype for P·V, as the
 *   reference's tl.dot; 16-byte aligned rows), everything else on CUDA cores in fp32; the
 *   backward as dsalt_attention_bwd. w_cont [T] fp32: the
 *   continuous window widths w̃. lmk [n_heads, n_seqs, k_lmk] int32 positions (one set per
 *   sequence, any slot order, -1 = none) and lmk_logw [n_heads, n_seqs, k_lmk] fp32 their
 *   log-weights log σ(s/τ_lmk). Query i attends to the band 0 <= i - j <= w̃(i) with the soft
 *   edge log σ((w̃ - (i - j)) / tau_win) outside the core i - j <= w̃ - win_edge, and to the
 *   landmarks p < i - w̃, p <= i with logit + log-weight. Forward: out [T, n_heads, head_dim]
 *   in out_dtype, lse [T, n_heads] (natural log; nullable); workspace from
 *   dsalt_train_attention_fwd_workspace_bytes. Backward (workspace from
 *   dsalt_attention_bwd_workspace_bytes): from out, dout and lse, writes dq, dk, dv
 *   (fp32, as dsalt_attention_bwd), d_logw [n_heads, n_seqs, k_lmk] and d_w [T] (the
 *   gradient of w̃, summed over heads); dk, dv, d_logw and d_w accumulate with atomic adds.
 */
size_t dsalt_train_attention_fwd_workspace_bytes(int64_t T, int n_heads, int n_seqs, int k_lmk);
int dsalt_train_attention_fwd(const void* q, const void* k, const void* v, int dtype, int64_t T, int n_heads,
                              int n_kv, int head_dim, int64_t q_stride, int64_t kv_stride, const float* w_cont,
                              const int32_t* lmk, const float* lmk_logw, int k_lmk, const int32_t* cu_seqlens,
                              int n_seqs, float tau_win, float win_edge, void* out, int out_dtype, float* lse,
                              void* workspace, size_t workspace_bytes, void* stream);
int dsalt_train_attention_bwd(const void* q, const void* k, const void* v, int dtype, int64_t T, int n_heads, int n_kv,
                              int head_dim, int64_t q_stride, int64_t kv_stride, const void* out, int out_dtype,
                              const void* dout, int dout_dtype, const float* lse, const float* w_cont,
                              const int32_t* lmk, const float* lmk_logw, int k_lmk, const int32_t* cu_seqlens,
                              int n_seqs, float tau_win, float win_edge, float* dq, float* dk, float* dv,
                              float* d_logw, float* d_w, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Sequence-sharded forms (no counterpart in the reference, which runs on one GPU): one
 * rank's share of a single sequence of seq_len positions split across ranks.
 *
 * dsalt_select_block_range: the block-causal sets [set_lo, set_hi) of one sequence whose
 *   signals (xnorm, vnorm, w: every position of the sequence, e.g. all-gathered from the
 *   ranks) are given; only the prefix [0, set_hi * block) is read. Same sets as
 *   dsalt_select_landmarks(DSALT_SELECT_BLOCK_CAUSAL) for those blocks. lmk_out
 *   [n_heads, set_hi - set_lo, k].
 * dsalt_attention_fwd_sharded: queries = positions [q_pos0, q_pos0 + q_rows) (q, out,
 *   lse rows 0..q_rows-1); k/v (this GPU's memory: they are read by TMA tile loads; only
 *   lmk_k_src / lmk_v_src may point to other GPUs) rows = positions [kv_pos0, kv_pos0 + kv_rows), which must
 *   hold every window key of the local queries (kv_pos0 <= q_pos0 - max width + 1; keys
 *   below kv_pos0 read as zero); w [seq_len] widths by position; lmk [n_heads,
 *   n_local_sets, k_lmk] positions within the sequence (one set per lmk_block local
 *   queries, or one set when lmk_block = 0), ascending, -1 last. Landmark rows are read
 *   from lmk_k_src[r] / lmk_v_src[r] (device arrays of pointers; rank r holds positions
 *   [r * rows_per_src, (r+1) * rows_per_src) with the kv token stride), which may be other
 *   GPUs' memory mapped by dsalt_ipc_open (plain NVLink loads), gathered once per call into
 *   the workspace as 128-row tiles. q_pos0 and q_rows are multiples of 128 (and of
 *   lmk_block); bf16 / fp16 inputs; head_dim 64 or 128.
 * dsalt_ipc_export / dsalt_ipc_open / dsalt_ipc_close: CUDA IPC handles (64 bytes) of a
 *   device pointer inside an allocation, for the peer tables above.
 */
size_t dsalt_select_block_range_workspace_bytes(int64_t seq_len, int n_heads, int n_kv, int k, int block,
                                                int set_hi);
int dsalt_select_block_range(const float* xnorm, const float* vnorm, const int32_t* w, const float* alpha,
                             int64_t seq_len, int n_heads, int n_kv, int k, int block, int set_lo, int set_hi,
                             int32_t* lmk_out, void* workspace, size_t workspace_bytes, void* stream);
size_t dsalt_attention_sharded_workspace_bytes(int64_t q_rows, int n_heads, int k_lmk, int lmk_block, int head_dim);
/* dsalt_select_shard: the block-causal sets of rank `rank`'s blocks, with the selection's
 *   per-chunk work spread over the ranks (no counterpart in the reference; same sets as
 *   dsalt_select_landmarks(DSALT_SELECT_BLOCK_CAUSAL) on the whole sequence, i.e. as
 *   results/causal_landmark_check.py:82-113 per block). The sequence of seq_len positions
 *   splits into n_ranks contiguous shards of seq_len / n_ranks positions, a whole number
 *   of blocks each; rank r owns blocks (= chunks = sets) [r * cpr, (r + 1) * cpr).
 *   xnorm [seq_len], vnorm [seq_len, n_kv], w [seq_len]: whole-sequence arrays of which
 *   phases 1-3 read only the own shard; phase 4 reads earlier positions as well when some
 *   alpha lies outside [0, 1] (no dominance pruning then), so gather the signals first in
 *   that case. workspace (dsalt_select_shard_workspace_bytes, the same size on every
 *   rank); peer_workspaces: device array of the n_ranks ranks' workspace pointers (own
 *   entry included; peers mapped by dsalt_ipc_open). Call phases 1, 2, 3, 4 in order with
 *   a cross-GPU barrier (dsalt_peer_barrier) between consecutive phases: 1 chunk sums of
 *   the own blocks; 2 reads the others' sums, prefix statistics, dominance grids of the
 *   own blocks; 3 reads the earlier ranks' grid totals, survivors of the own blocks; 4
 *   reads the earlier ranks' survivors and writes lmk_out [n_heads, cpr, k]. A rank's
 *   workspace must not be reused before every rank has finished phase 4. n_kv <= 32. */
size_t dsalt_select_shard_workspace_bytes(int64_t seq_len, int n_heads, int n_kv, int k, int block);
int dsalt_select_shard(int phase, const float* xnorm, const float* vnorm, const int32_t* w, const float* alpha,
                       int64_t seq_len, int n_heads, int n_kv, int k, int block, int rank, int n_ranks,
                       void* workspace, size_t workspace_bytes, const void* const* peer_workspaces, int32_t* lmk_out,
                       void* stream);
int dsalt_attention_fwd_sharded(const void* q, const void* k, const void* v, int dtype, int64_t q_rows, int n_heads,
                                int n_kv, int head_dim, int64_t q_stride, int64_t kv_stride, int64_t q_pos0,
                                int64_t kv_pos0, int64_t kv_rows, int64_t seq_len, const int32_t* w,
                                const int32_t* lmk, const float* lmk_bias, int k_lmk, int lmk_block,
                                const void* const* lmk_k_src, const void* const* lmk_v_src, int64_t rows_per_src,
                                void* out, int out_dtype, float* lse, void* workspace, size_t workspace_bytes,
                                void* stream);
/* dsalt_peer_barrier: rank `rank` of n_ranks GPUs (one process each) stores `epoch` in its
 *   own flag (an int in its memory) and waits until every rank's flag (peer_flags: device
 *   array of the ranks' flag pointers, peers mapped by dsalt_ipc_open) has reached it;
 *   epochs must increase from call to call. epoch <= 0 takes the epoch from a device-side
 *   counter in own_flag[1] (incremented by the call; own_flag then points to two ints), so
 *   that a CUDA graph holding the call advances it on every replay. Memory written on this GPU before the call is
 *   visible to the peers' work queued after theirs. A wait longer than 2 s gives up and
 *   sets the device status word (no hang).
 * dsalt_peer_allgather: dst[j * bytes_per_rank ...] <- src[j][0 .. bytes_per_rank) for
 *   every rank j != rank (src: device array of the ranks' pointers; 16-byte multiples).
 * dsalt_peer_copy: bytes from src (this or a peer GPU's memory) to dst, on the stream. */
int dsalt_peer_barrier(int* own_flag, const int* const* peer_flags, int n_ranks, int rank, int epoch, void* stream);
int dsalt_peer_allgather(void* dst, const void* const* src, int n_ranks, int rank, int64_t bytes_per_rank,
                         void* stream);
int dsalt_peer_copy(void* dst, const void* src, int64_t bytes, void* stream);
int dsalt_ipc_export(const void* ptr, void* handle_out, int64_t* offset_out);
int dsalt_ipc_open(const void* handle, int64_t offset, void** ptr_out);
int dsalt_ipc_close(void* ptr, int64_t offset);

/*
 * dsalt_attention_fwd without a workspace: no counterpart in the reference.
 * For callers that cannot allocate device memory: a host binding that holds only the
 * caller's q/k/v/out pointers and no device allocator of its own (a cgo, JNI or ctypes
 * binding with no framework behind it), or a serving loop whose memory pool is fully
 * reserved for its caches and may not grow between requests. The scratch that
 * dsalt_attention_fwd takes from `workspace` (two sequence tables of n_seqs+1 int32 and a
 * 32-byte plan per 128-query tile) comes here from a static device array of this library
 * (417 KB), one per device:
 *   - at most DSALT_NOALLOC_MAX_SEQS sequences and DSALT_NOALLOC_MAX_TOKENS tokens;
 *     larger requests fail with DSALT_ERR_UNSUPPORTED before any work is queued;
 *   - nothing in it needs to start at zero: each call rewrites the tables it reads;
 *   - every call on a device shares it, so calls that may overlap on one device (other
 *     streams, other host threads) race on it; the caller serialises them;
 *   - the first call on each device looks the array's address up (cudaGetSymbolAddress);
 *     make that first call before any stream capture begins.
 * Nothing is allocated (no cudaMalloc, no allocating library). Arguments, results and
 * error codes are otherwise those of dsalt_attention_fwd (the same kernels run).
 */
#define DSALT_NOALLOC_MAX_SEQS 4096
#define DSALT_NOALLOC_MAX_TOKENS 1048576
int dsalt_attention_fwd_noalloc(const void* q, const void* k, const void* v, int dtype, int64_t T, int n_heads,
                                int n_kv, int head_dim, int64_t q_stride, int64_t kv_stride, const int32_t* w,
                                const int32_t* lmk, const float* lmk_bias, int k_lmk, int lmk_block,
                                const int32_t* cu_seqlens, int n_seqs, int max_seqlen, void* out, int out_dtype,
                                float* lse, void* stream);

/*
 * The whole inference core of DSALTAttention._packed after the projections and RoPE
 * (dsalt/modules/dsalt_attention.py:610-625): widths, signals, selection, attention.
 * Scratch for the intermediates comes from `workspace`
 * (dsalt_core_workspace_bytes); w_out / lmk_out (nullable) receive copies of the widths
 * and landmark sets; logit_in (nullable) is dsalt_token_signals' caller-computed logit.
 */
size_t dsalt_core_workspace_bytes(int mode, int64_t T, int n_seqs, int max_seqlen, int n_heads, int n_kv,
                                  int head_dim, int k, int block);
int dsalt_core_forward(int mode, const void* x, int x_dtype, int d_model, int64_t x_stride, const void* gate_w,
                       const void* gate_b, int gate_dtype, const void* logit_in, int n_min, int n_max,
                       const float* alpha, int norm_mode, const void* q, const void* k, const void* v, int qkv_dtype, int n_heads,
                       int n_kv, int head_dim, int64_t q_stride, int64_t kv_stride, int k_lmk, int block,
                       const int32_t* cu_seqlens, int n_seqs, int64_t T, int max_seqlen, void* out, int out_dtype,
                       int32_t* w_out, int32_t* lmk_out, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Serving operators (no counterpart in the reference, which recomputes the whole sequence
 * for every token): a paged key/value cache in 8 bits, the attention that reads it, and
 * sampling. Lengths, tables and counts are device data, so a captured call follows them.
 *
 * Pages hold page_size tokens (16, 32, 64 or 128) of every kv head. block_tables
 * [n_seqs, max_pages] int32 lists the pages of each row (sequence), -1 where none; the pages
 * of no row are a stack free_pages [free_capacity] of which the first n_free [1] count.
 *
 * dsalt_reserve_slots: pages and slots for new_lens [n_seqs] more tokens of rows that hold
 *   seq_lens [n_seqs] (negative numbers count as 0). Tokens are packed row after row;
 *   n_tokens is the room in slots / positions. A row is granted when its table
 *   (max_pages * page_size tokens) and the room hold its new tokens and either it needs no
 *   page or the running sum of needed pages, over the rows that fit in order, is at most
 *   n_free; a row that is not granted keeps its length and gets nothing. Page number j of
 *   that order is free_pages[n_free - 1 - j]. Writes the new table entries, slots [n_tokens]
 *   int64 (page * page_size + offset; -1 for tokens of rows not granted and behind the last
 *   token), positions [n_tokens] (0 there), cu_new [n_seqs + 1] (first token of each row,
 *   at most n_tokens), granted [n_seqs] bytes, seq_lens_out and n_free_out (which may be
 *   seq_lens and n_free). At most 8192 rows. slots and positions 16-byte aligned.
 * dsalt_release_slots: gives the pages of the rows flagged in release [n_seqs] bytes back to
 *   the stack, in the order in which reserve would take them again; their entries become -1
 *   and their lengths 0. A page in the tables of two flagged rows is given back twice.
 */
int dsalt_reserve_slots(int32_t* block_tables, int n_seqs, int max_pages, const int32_t* seq_lens,
                        const int32_t* new_lens, const int32_t* free_pages, int64_t free_capacity,
                        const int32_t* n_free, int page_size, int64_t n_tokens, int64_t* slots, int32_t* positions,
                        int32_t* cu_new, uint8_t* granted, int32_t* seq_lens_out, int32_t* n_free_out, void* stream);
int dsalt_release_slots(int32_t* block_tables, int n_seqs, int max_pages, int32_t* seq_lens, const uint8_t* release,
                        int32_t* free_pages, int64_t free_capacity, int32_t* n_free, int page_size, void* stream);

/*
 * dsalt_append_cache: quantises the keys and values of T new tokens into their slots.
 * k, v [T, n_kv, head_dim] of dtype (token and head strides in elements; 16-byte aligned
 *   rows; head_dim 64 or 128); k_cache, v_cache [n_pages, n_kv, page_size, head_dim] e4m3
 *   bytes; k_scale, v_scale [n_pages, n_kv] fp32, powers of two: an element is byte * scale.
 * The scale of a (page, kv head) is the smallest 2^e, e >= -110, with amax <= 448 * 2^e over
 *   the tokens of the page; it starts afresh in a call that writes the page's first token,
 *   otherwise it never falls, and when it grows the bytes already there are rescaled (rounded
 *   to nearest even). Infinities are stored as the largest value (448 * 2^e) and do not count
 *   for amax, NaN as NaN.
 * slots [T] int64; negative or beyond the pool: the token is left out. The slots of one page
 *   must be distinct and lie within page_size consecutive tokens of the call, in any order (as
 *   dsalt_reserve_slots numbers them: next to each other).
 */
int dsalt_append_cache(const void* k, const void* v, int dtype, int64_t T, int n_kv, int head_dim,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                       void* k_cache, void* v_cache, float* k_scale, float* v_scale, int64_t n_pages, int page_size,
                       const int64_t* slots, void* stream);

/*
 * dsalt_cache_attention: attention of the last query tokens of each sequence over the cache.
 * q [T, n_heads, head_dim] (token stride q_stride, 16-byte aligned rows; bf16, fp16 or fp32;
 *   head_dim 64 or 128); cache, scales and tables as above; head h reads kv head
 *   h / (n_heads / n_kv).
 * seq_lens [n_seqs]: tokens in the cache, the query tokens included; cu_q [n_seqs + 1]
 *   (starting at 0, at most T): query tokens of each sequence, the r-th of n at position
 *   seq_len - n + r. Null: one per sequence, T = n_seqs.
 * w [T] int32 widths (at least 1 is taken): the query at position i attends to
 *   [max(0, i - w + 1), i] and to the landmarks lmk [n_heads, n_seqs, k_lmk] p with
 *   0 <= p < i - w + 1 (any order, distinct, -1 = none), whose logits get lmk_bias (nullable).
 *   w null: to [0, i], k_lmk = 0.
 * k_scale, v_scale: any positive numbers (dsalt_append_cache writes powers of two), or 0.
 * out [T, n_heads, head_dim] in out_dtype, lse [T, n_heads] (nullable, natural log). A query
 *   without keys and rows behind cu_q's last token give zeros and -inf.
 * Keys on a page number outside [0, n_pages) are left out and reported in the device status
 *   word. Deterministic. At most 8192 sequences.
 */
size_t dsalt_cache_attention_workspace_bytes(int64_t T, int n_seqs, int n_heads, int n_kv, int head_dim);
int dsalt_cache_attention(const void* q, int dtype, int64_t T, int n_heads, int n_kv, int head_dim, int64_t q_stride,
                          const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                          int64_t n_pages, int page_size, const int32_t* block_tables, int max_pages,
                          const int32_t* seq_lens, int n_seqs, const int32_t* cu_q, const int32_t* w,
                          const int32_t* lmk, const float* lmk_bias, int k_lmk, void* out, int out_dtype, float* lse,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * dsalt_sample: one token per row of logits [B, V] (row stride in elements, any alignment;
 * fp32, bf16 or fp16; V at most 2^20) from given uniforms u [B] in [0, 1).
 * With weights exp((l - max l) / temperature): top_k keeps the k first in the order (logit
 *   descending, index ascending), top_p of those the shortest prefix whose mass reaches top_p
 *   times theirs, min_p of those the weights of at least min_p; token is the first index
 *   whose running sum of kept weights (index order) exceeds u times their total, logprob
 *   (nullable) log of its share of that total.
 * Each setting is a device array [B], or null and the value beside it. temperature <= 0 takes
 *   the first index of the largest logit (logprob 0); top_k outside [1, V), top_p >= 1 and
 *   min_p <= 0 are off; of a min_p above 1, which no weight reaches, the first of the order stays.
 *   A NaN logit counts as -inf; +inf logits share the draw; a row of
 *   nothing but -inf gives token 0 and logprob -inf.
 */
int dsalt_sample(const void* logits, int dtype, int64_t B, int64_t V, int64_t row_stride, const float* u,
                 const float* temperature, float temperature_value, const int32_t* top_k, int top_k_value,
                 const float* top_p, float top_p_value, const float* min_p, float min_p_value, int64_t* token,
                 float* logprob, void* stream);

/*
 * What a decoder block computes around its attention.
 *
 * dsalt_pack8, dsalt_unpack8: activations in 8 bits. Of a row, 32 neighbouring values (the last
 *   group may be shorter) share the scale 2^(s - 127), kept as the byte s; a value is code *
 *   2^(s - 127) with code = clamp(rint(x * 2^(127 - s)), -127, 127), s = max(E - 6, 1), E the fp32
 *   exponent field of the group's largest magnitude. A group with a NaN or an infinity gets s = 255
 *   and reads as NaN as a whole.
 * x [rows, cols] of dtype (row stride in elements), codes [rows, cols] int8, exps
 *   [rows, ceil(cols / 32)] bytes, out [rows, cols] contiguous (rounded to nearest even where its
 *   type holds fewer bits).
 */
int dsalt_pack8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* codes, uint8_t* exps,
                void* stream);
int dsalt_unpack8(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* out, int dtype,
                  void* stream);

/*
 * dsalt_qk_norm_rope: per head, RMS norm with a weight per channel (q_weight, k_weight [head_dim] of
 * w_dtype; both null: no norm), then the half-split rotation by the token's angles.
 * q [T, n_heads, head_dim], k [T, n_kv, head_dim] of dtype (token and head strides in elements;
 *   16-byte aligned rows), q_out and k_out contiguous. head_dim a multiple of 16 (fp32: 8) up to 256.
 * cos, sin [table_rows, at least head_dim / 2] fp32 (row stride table_stride, 16-byte aligned rows);
 *   the angles of the first half's channels are read, the second half turns by the same. Token t
 *   takes row positions[t], or row t where positions is null. A position outside the tables is
 *   reported in the device status word (51) and taken as 0. At most 4096 heads, and 2^30 groups of up to
 *   four heads (forward) or two (backward).
 * dsalt_qk_norm_rope_bwd: gradients of q, k (contiguous, of dtype) and of the weights (of w_dtype)
 *   from those of the outputs, dq_out and dk_out (token and head strides as above). Deterministic.
 */
int dsalt_qk_norm_rope(const void* q, const void* k, int dtype, int64_t T, int n_heads, int n_kv, int head_dim,
                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                       const void* q_weight, const void* k_weight, int w_dtype, float eps, const float* cos,
                       const float* sin, int64_t table_rows, int64_t table_stride, const int32_t* positions, void* q_out,
                       void* k_out, void* stream);
size_t dsalt_qk_norm_rope_bwd_workspace_bytes(int head_dim);
int dsalt_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, int dtype, int64_t T,
                           int n_heads, int n_kv, int head_dim, int64_t q_token_stride, int64_t q_head_stride,
                           int64_t k_token_stride, int64_t k_head_stride, int64_t dq_token_stride,
                           int64_t dq_head_stride, int64_t dk_token_stride, int64_t dk_head_stride,
                           const void* q_weight, const void* k_weight, int w_dtype, float eps, const float* cos,
                           const float* sin, int64_t table_rows, int64_t table_stride, const int32_t* positions,
                           void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace,
                           size_t workspace_bytes, void* stream);

/*
 * dsalt_gated_ffn: y = (act(x Wg^T) * (x Wu^T)) Wd^T.
 * x [T, d_model] of dtype (row stride x_stride), w_gate, w_up [d_ff, d_model], w_down [d_out, d_ff], y
 *   [T, d_out], contiguous, all of dtype. The product of gate and up is rounded to dtype before the
 *   last product; sums are fp32. activation: DSALT_ACT_SILU, or DSALT_ACT_GELU (by the error function).
 * keep: what the backward pass needs goes to kept, in rows of pitch = dsalt_gated_ffn_pitch(d_ff) values, a
 *   multiple of 32. DSALT_KEEP_INPUT: [3, T, pitch] of dtype's size: of fp32 x Wg^T, x Wu^T and the product's
 *   rows; of 16-bit types the upper halves of x Wg^T and of x Wu^T in fp32, then the third byte of each (an up's behind
 *   its gate's), so that every value is held to 2^-15 of itself (kept_exps must be given here too; nothing
 *   is written there). DSALT_KEEP_8BIT: [2, T, pitch] bytes, x Wg^T and x Wu^T as codes with scales in
 *   kept_exps [2, pitch / 32, T], as dsalt_pack8 forms them. kept and workspace 256-byte aligned.
 * dsalt_gated_ffn_bwd: the gradients (contiguous, of dtype; null: not wanted, dw_gate and dw_up go
 *   together) from dy [T, d_out] (row stride dy_stride). With DSALT_KEEP_8BIT x holds the codes and
 *   x_exps the scales of dsalt_pack8 (contiguous), else x is the forward's. x may be null where dw_gate is.
 * 16-bit types whose sizes are multiples of 8 run on the tensor cores (operands and their rows 16-byte
 *   aligned), everything else on the CUDA cores. Deterministic.
 */
#define DSALT_ACT_SILU 0
#define DSALT_ACT_GELU 1
#define DSALT_KEEP_NONE 0
#define DSALT_KEEP_INPUT 1
#define DSALT_KEEP_8BIT 2
int64_t dsalt_gated_ffn_pitch(int d_ff);
size_t dsalt_gated_ffn_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out);
/* with what is kept: DSALT_KEEP_INPUT of fp32 needs almost none */
size_t dsalt_gated_ffn_keep_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out, int keep);
int dsalt_gated_ffn(const void* x, int dtype, int64_t T, int d_model, int64_t x_stride, const void* w_gate,
                    const void* w_up, const void* w_down, int d_ff, int d_out, int activation, int keep, void* kept,
                    uint8_t* kept_exps, void* y, void* workspace, size_t workspace_bytes, void* stream);
size_t dsalt_gated_ffn_bwd_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out, int keep);
int dsalt_gated_ffn_bwd(const void* dy, int dtype, int64_t T, int d_model, int64_t dy_stride, const void* x,
                        int64_t x_stride, const uint8_t* x_exps, const void* w_gate, const void* w_up,
                        const void* w_down, int d_ff, int d_out, int activation, int keep, const void* kept,
                        const uint8_t* kept_exps, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* workspace,
                        size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSALT_B200_H */
