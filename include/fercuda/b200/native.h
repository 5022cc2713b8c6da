/*
 * Native launchers of libptx_kernels.so beyond the reference's tensor-op ABI.
 * No reference counterpart: these are the kernels the session layer
 * (libfercuda_capi.so) and the transformer driver call, exported so C/C++
 * callers that manage their own device memory can use them directly.
 *
 * Every launcher queues work on `stream` and returns without synchronising;
 * a non-cudaSuccess return means nothing was launched (argument errors are
 * cudaErrorInvalidValue, shapes a kernel does not take cudaErrorNotSupported).
 * `err` (may be null) is a device word the kernels OR error bits into:
 * 1 a bulk copy did not land within about one second, 2 a tensor-core commit
 * did not arrive in time, 4 a shape the kernel cannot take, 8 a producer /
 * consumer hand-off timed out.
 */
#ifndef FERCUDA_B200_NATIVE_H
#define FERCUDA_B200_NATIVE_H

#include <stddef.h>
#include <stdint.h>

#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- GEMM on the tensor cores (tcgen05) ------------------------------------
 * C[M,N] = A[M,K] . B[K,N], A and B row-major bf16, f32 accumulation, fixed K
 * order, no split-K: bit-identical run to run. K % 8 == 0, N % 8 == 0, all
 * pointers 16-byte aligned.
 * epi: 0 C f32; 1 C bf16; 2 C bf16 = GELU(acc) (erf form); 3 C f32 =
 * resid + acc (resid == c adds in place; another resid is copied into c first
 * and must not partly overlap it). */
cudaError_t fer_gemm_bf16_tc_ex(const void* a, const void* b, void* c, const float* resid, int M, int N, int K,
                                int epi, uint32_t* err, cudaStream_t stream);
/* out_dtype: 0 f32, 2 bf16 (fer_buffer_dtype_t codes). */
cudaError_t fer_gemm_bf16_tc(const void* a, const void* b, void* c, int M, int N, int K, uint32_t out_dtype,
                             uint32_t* err, cudaStream_t stream);
/* Split-K form for short M (decode steps): K split into ranges of 64-deep
 * blocks computed by separate CTAs, partials added in range order before
 * `epi` (for epi 3 the residual is c). Deterministic; the additions are
 * grouped differently from fer_gemm_bf16_tc_ex.
 * splits <= 0: cluster form, one cluster of fer_gemm_splitk_cluster_splits()
 * CTAs per output tile adding the partials through distributed shared memory
 * in one kernel (ws unused), or the single-pass kernel when that is 1.
 * splits > 0 (or FERCUDA_SPLITK_CLUSTER=0): partials in the f32 workspace
 * `ws`, added by a second kernel; the count is reduced to fit ws_bytes.
 * Both forms give the same bits for the same split count.
 * flags bit 0: b is not written by the kernel just before this call on the
 * stream (weights); its first tiles are then fetched before the programmatic
 * launch wait, overlapping that kernel.
 * fer_gemm_splitk_workspace_bytes: ws for the workspace form's automatic count. */
size_t fer_gemm_splitk_workspace_bytes(int M, int N, int K);
int fer_gemm_splitk_cluster_splits(int M, int N, int K);
cudaError_t fer_gemm_bf16_tc_splitk(const void* a, const void* b, void* c, int M, int N, int K, int epi, int splits,
                                    float* ws, size_t ws_bytes, int flags, uint32_t* err, cudaStream_t stream);
/* 0 (default): 2-CTA cluster kernel for M > 128; 1: single-CTA kernel. Both
 * give the same bits. Process-wide. */
void fer_gemm_tc_set_mode(int mode);
/* 2-CTA clusters the GEMM launches at most (-1 before its first 2-CTA call). */
int fer_gemm_tc_clusters(void);

/* ---- reference-order matmul (CUDA cores) ----------------------------------
 * One sequential fmaf chain over K per output, the reference k_matmul_f32
 * order (src/runtime/ops_bridge.cu:13-31). dtype: fer_buffer_dtype_t of all
 * three matrices (f32, f16, bf16, i8, u8; computed in f32). */
cudaError_t fer_matmul_ref_order(const void* a, const void* b, void* c, int M, int K, int N, uint32_t dtype,
                                 cudaStream_t stream);
cudaError_t fer_matmul_bf16_f32_ref_order(const void* a, const void* b, float* c, int M, int K, int N,
                                          cudaStream_t stream);
/* Element casts used by the session layer's staging (dtype as above). */
cudaError_t fer_cast_to_f32(const void* in, float* out, size_t n, uint32_t dtype, cudaStream_t s);
cudaError_t fer_cast_from_f32(const float* in, void* out, size_t n, uint32_t dtype, cudaStream_t s);

/* ---- row kernels -------------------------------------------------------------
 * flags: 1 softmax, 2 layer norm, 3 softmax then layer norm; gamma / beta
 * optional [cols] f32. fer_rows_f32: bit-identical to the reference kernels.
 * fer_rows_fast_f32: deterministic, within 1e-5 of the largest output of the
 * reference order; cudaErrorNotSupported for cols % 4 != 0, cols > 8192,
 * in-place or unaligned buffers. fer_rows_f32_pdl / fer_rows_fast_f32_pdl:
 * the same launched
 * with programmatic dependent launch; early 1 lets the first loads,
 * early 2 the whole kernel run before it waits for the kernel just before it
 * on the stream (the caller promises that kernel writes none of x / gamma /
 * beta, and for 2 that it neither reads nor writes y). */
cudaError_t fer_rows_f32(const float* x, float* y, const float* gamma, const float* beta, int rows, int cols,
                         float eps, uint32_t flags, uint32_t* err, cudaStream_t stream);
cudaError_t fer_rows_f32_pdl(const float* x, float* y, const float* gamma, const float* beta, int rows, int cols,
                             float eps, uint32_t flags, uint32_t early, uint32_t* err, cudaStream_t stream);
cudaError_t fer_rows_fast_f32(const float* x, float* y, const float* gamma, const float* beta, int rows, int cols,
                              float eps, uint32_t flags, uint32_t* err, cudaStream_t stream);
cudaError_t fer_rows_fast_f32_pdl(const float* x, float* y, const float* gamma, const float* beta, int rows, int cols,
                                  float eps, uint32_t flags, uint32_t early, uint32_t* err, cudaStream_t stream);
/* Layer norm of every row of x [rows, cols] (no affine) for any buffer dtype
 * (fer_buffer_dtype_t): computed in f32 in the reference order, each value
 * widened on load and rounded back on store as the reference's cast staging
 * does (src/runtime/exec_planner.cu:304-387), so the bits equal cast ->
 * fer_rows_f32 -> cast; one launch, no temporaries; x == y allowed. f32 runs
 * fer_rows_f32. */
cudaError_t fer_layer_norm_typed(const void* x, void* y, int rows, int cols, float eps, uint32_t dtype,
                                 uint32_t* err, cudaStream_t stream);

/* ---- intents -------------------------------------------------------------------
 * Deterministic sum / max of n floats into out[0] (sum adds to out[0], as the
 * reference's atomics do); scratch holds fer_reduce_scratch_floats(n) floats. */
size_t fer_reduce_scratch_floats(unsigned int n);
cudaError_t fer_reduce_f32(const float* in, float* out, float* scratch, unsigned int n, int is_max, cudaStream_t s);
/* Direct 2-D convolution: input [H, W, C], weights [F, C, KH, KW], output
 * [out_h, out_w, F]; optional bias [F] and relu. */
cudaError_t fer_conv2d_f32(const float* input, const float* weights, const float* bias, float* output,
                           unsigned int H, unsigned int W, unsigned int C, unsigned int KH, unsigned int KW,
                           unsigned int F, unsigned int pad_h, unsigned int pad_w, unsigned int sh, unsigned int sw,
                           int relu, cudaStream_t s);

/* ---- transformer building blocks ------------------------------------------------
 * Causal attention, head_dim 64, from the fused activation qkv [B*S, 3d]
 * (q | k | v, head h at columns 64h of each third) into out [B*S, d], bf16.
 * flags bit 0 forces the mma.sync kernel; otherwise S % 128 == 0 takes the
 * tcgen05 kernel. fer_attn_causal == fer_attn_causal_ex(..., 0, NULL, s). */
cudaError_t fer_attn_causal_ex(const void* qkv, void* out, int B, int S, int d, int heads, int flags, uint32_t* err,
                               cudaStream_t s);
cudaError_t fer_attn_causal(const void* qkv, void* out, int B, int S, int d, int heads, cudaStream_t s);
/* The tcgen05 kernel alone: cudaErrorNotSupported where it does not apply. */
cudaError_t fer_attn_causal_tc(const void* qkv, void* out, int B, int S, int d, int heads, uint32_t* err,
                               cudaStream_t stream);
/* KV cache (per layer [max_batch][heads][max_seq][64] bf16, K and V blocks):
 * fer_kv_store copies the K and V parts of qkv [B*S, 3d] (rows b*S + s) to
 * positions pos0 + s of sequences b. fer_attn_decode: one query per sequence
 * (the Q part of row b of qkv_dec [B, 3d]) against positions 0 .. n_keys-1,
 * out [B, d] bf16; split into 256-position chunks combined in chunk order,
 * scratch of fer_attn_decode_scratch_floats(B, heads, n_keys) floats (0: none
 * needed). head_dim 64. err: optional device error word (bulk-copy wait
 * timeouts). */
cudaError_t fer_kv_store(const void* qkv, void* k_cache, void* v_cache, int B, int S, int d, int heads, int max_seq,
                         int pos0, cudaStream_t s);
size_t fer_attn_decode_scratch_floats(int B, int heads, int n_keys);
cudaError_t fer_attn_decode(const void* qkv_dec, const void* k_cache, const void* v_cache, void* out, float* scratch,
                            int B, int d, int heads, int max_seq, int n_keys, uint32_t* err, cudaStream_t s);
/* The decode step's cache store + attention in one kernel, with the position
 * in device memory (*d_len = position of the new token, advanced by the
 * caller with fer_device_int_add): launch arguments never change between
 * steps, so the step can be captured in a CUDA graph and replayed. scratch
 * as fer_attn_decode_scratch_floats(B, heads, max_seq); counters: B * heads
 * ints, zero before the first call and left zero by every call. */
cudaError_t fer_decode_kv_attention(const void* qkv_dec, void* k_cache, void* v_cache, void* out, float* scratch,
                                    int* counters, int B, int d, int heads, int max_seq, int* d_len, uint32_t* err,
                                    cudaStream_t s);
cudaError_t fer_device_int_add(int* d_len, int v, cudaStream_t s);
cudaError_t fer_device_int_set(int* d_len, int v, cudaStream_t s);
/* ---- rotary positions -------------------------------------------------------------
 * Rotates the first rotary_dim elements of each of `heads` heads of every row
 * of x [rows, heads * head_dim] (rows x_stride elements apart) into out (rows
 * out_stride apart; out == x with equal strides rotates in place, other
 * overlaps are not allowed); the rest of a head is copied. Pair i (i <
 * rotary_dim / 2) is elements (i, i + rotary_dim / 2) of the head, or (2i,
 * 2i + 1) with FER_ROTARY_FLAG_INTERLEAVED; it turns by positions[row][axis]
 * * base^-e. Pairs are dealt to the axes in order, sections[a] each
 * (sections add up to rotary_dim / 2); e = i / (rotary_dim / 2), or with
 * FER_ROTARY_FLAG_AXIS_FREQS j / sections[axis] for the j-th pair of its
 * axis. FER_ROTARY_FLAG_INVERSE turns back: the inverse, and the gradient.
 * Angles are reduced in 64 bits, products are f32, rounded once to the
 * output. dtype: fer_buffer_dtype_t f32, f16 or bf16. */
#define FER_ROTARY_FLAG_INTERLEAVED 1u
#define FER_ROTARY_FLAG_AXIS_FREQS 2u
#define FER_ROTARY_FLAG_INVERSE 4u
typedef struct fer_rotary_args {
    const void* x;
    void* out;
    const int32_t* positions;    /* [rows, axes] */
    size_t x_stride, out_stride; /* elements */
    int rows, heads, head_dim, rotary_dim, axes;
    int sections[4];
    float base;
    uint32_t flags;
    uint32_t dtype;
} fer_rotary_args_t;
cudaError_t fer_rotary(const fer_rotary_args_t* args, cudaStream_t s);

/* Root-mean-square norm of each head and its rotary positions in one pass, as
 * fer_rotary with flags INTERLEAVED and AXIS_FREQS only and head_dim at most 256:
 * a head x becomes x / sqrt(mean(x^2) + eps) * gamma over all of its elements,
 * then its first rotary_dim elements turn. The first heads - k_heads heads take
 * q_gamma, the last k_heads k_gamma, f32 [head_dim] each (NULL: ones). f32
 * inside, rounded once. eps >= 0.
 * fer_norm_rotary_grad: rotary.x is the call's x, grad the gradient of its out
 * (grad_stride elements apart), rotary.out receives the gradient of x (out ==
 * grad or out == x with equal strides is allowed), q_gamma_grad / k_gamma_grad
 * (NULL: not wanted) those of the gammas, summed over rows and heads in a fixed
 * order. workspace: fer_norm_rotary_grad_workspace_bytes, 16-byte aligned, any
 * contents; calls (or graph replays) that may run at the same time need one each. */
typedef struct fer_norm_rotary_args {
    fer_rotary_args_t rotary;
    int k_heads;
    const float* q_gamma;
    const float* k_gamma;
    float eps;
} fer_norm_rotary_args_t;
typedef struct fer_norm_rotary_grad {
    const void* grad;
    size_t grad_stride;
    float* q_gamma_grad;
    float* k_gamma_grad;
    void* workspace;
    size_t workspace_bytes;
} fer_norm_rotary_grad_t;
size_t fer_norm_rotary_grad_workspace_bytes(int rows, int heads, int head_dim);
cudaError_t fer_norm_rotary(const fer_norm_rotary_args_t* args, uint32_t* err, cudaStream_t s);
cudaError_t fer_norm_rotary_grad(const fer_norm_rotary_args_t* args, const fer_norm_rotary_grad_t* grad, uint32_t* err,
                                 cudaStream_t s);

/* ---- paged key-value cache ----------------------------------------------------------
 * K and V in pages [pages][kv_heads][page_size][head_dim] (f16 or bf16, 16-byte
 * aligned); slot s of sequence b is row s % page_size of page
 * page_table[b][s / page_size], and slots 0 .. lengths[b] - 1 are held.
 * page_size is a power of two from 8 to 256, head_dim 64, 128 or 256. A page
 * id outside [0, pages), or a length outside [0, max_pages * page_size], that
 * a kernel meets sets error bit 4; the length is clamped, attention skips slots
 * of such a page (as if not held), store drops their rows and evict, which
 * selects among all slots, copies no row from or to one. Entries behind the last held slot are
 * not read. Pages that fer_paged_store or fer_paged_evict write belong to one
 * place of one sequence; fer_paged_attention only reads pages, which may be
 * shared. Arrays of 32-bit numbers start at multiples of 4 bytes. */
typedef struct fer_paged_view {
    void* k;
    void* v;
    const int32_t* page_table;   /* [batch, max_pages] */
    const int32_t* lengths;      /* [batch] */
    int batch, max_pages, pages, kv_heads, page_size, head_dim;
    uint32_t dtype;
} fer_paged_view_t;
/* Appends rows: sequence b < n_seq takes rows offsets[b] .. offsets[b+1] - 1
 * (offsets NULL: row b), its i-th row to slot lengths[b] + i. k_rows / v_rows
 * [rows, kv_heads * head_dim], k_stride / v_stride elements apart. Rows behind
 * offsets[n_seq] belong to nobody. new_lengths (may be the view's lengths)
 * receives the n_seq sequences' lengths after the call. Optional: weights f32
 * and positions i32, both [batch, kv_heads, max_pages * page_size], receive 0
 * and seen[b] + i for each new slot, and new_seen (may be seen) seen[b] + the
 * new rows. Rows that do not fit set error bit 4 and are dropped. */
typedef struct fer_paged_store_args {
    const void* k_rows;
    const void* v_rows;
    size_t k_stride, v_stride;
    int rows, n_seq;
    const int32_t* offsets;      /* [n_seq + 1] or NULL */
    int32_t* new_lengths;
    float* weights;              /* NULL: none */
    int32_t* positions;          /* NULL: none; else seen and new_seen are given */
    const int32_t* seen;
    int32_t* new_seen;
} fer_paged_store_args_t;
cudaError_t fer_paged_store(const fer_paged_view_t* cache, const fer_paged_store_args_t* args, uint32_t* err,
                            cudaStream_t s);
/* Attention of one query per sequence b < n_seq over its held slots, heads
 * (a multiple of kv_heads; consecutive heads share a key head) of q [n_seq,
 * heads * head_dim] (q_stride elements apart), into out (out_stride apart,
 * not overlapping q): softmax(scale q.k) v, f32 statistics, rounded once. lse
 * (optional) [n_seq, heads]: log of the sum of exp(scale q.k). weights
 * (optional) f32 [batch, kv_heads, max_pages * page_size]: each held slot's
 * probabilities, summed over the heads that share it in head order, are
 * added. A sequence of no slots gives zeros, lse -inf. Deterministic, and a
 * sequence's results do not depend on the others in the batch. workspace:
 * fer_paged_attention_workspace_bytes, 16-byte aligned, any contents; two
 * calls (or graph replays) that may run at the same time need one each. */
typedef struct fer_paged_attention_args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int n_seq, heads;
    float scale;                 /* up to 2e38; 0: 1 / sqrt(head_dim) */
    float* lse;
    float* weights;
    void* workspace;
    size_t workspace_bytes;
} fer_paged_attention_args_t;
size_t fer_paged_attention_workspace_bytes(int n_seq, int heads, int kv_heads, int head_dim, int max_slots,
                                           int with_weights);
cudaError_t fer_paged_attention(const fer_paged_view_t* cache, const fer_paged_attention_args_t* args, uint32_t* err,
                                cudaStream_t s);
/* Cuts every sequence of more than `budget` slots down to `budget`, for each
 * key head on its own. Kept are the slots whose position is at least
 * seen[b] - recent, then those of the largest weight (NaN is the least; ties
 * and a surplus of recent slots go to the lowest slot). Kept slots before
 * `budget` stay where they are, and the i-th kept slot behind it moves into
 * the i-th freed slot before it: its key, value, weight and position. new_*
 * (each may be the array it continues) receive the results; slots behind a
 * sequence's new length are left as they were. workspace:
 * fer_paged_evict_workspace_bytes, rules as above. */
typedef struct fer_paged_evict_args {
    int budget, recent;          /* 1 <= budget, 0 <= recent <= budget */
    const float* weights;
    const int32_t* positions;
    const int32_t* seen;         /* [batch] */
    int32_t* new_lengths;
    float* new_weights;
    int32_t* new_positions;
    void* workspace;
    size_t workspace_bytes;
} fer_paged_evict_args_t;
size_t fer_paged_evict_workspace_bytes(int batch, int kv_heads, int max_slots, int budget);
cudaError_t fer_paged_evict(const fer_paged_view_t* cache, const fer_paged_evict_args_t* args, uint32_t* err,
                            cudaStream_t s);
/* The plan of a step: sequence b < batch holds lengths[b] slots and asks for
 * counts[b] new rows; its row of page_table has held[b] pages. free_pages is a
 * ring of `pages` entries and free_state says where the free ones begin and how
 * many there are. Sequences are served in order: b gets its rows if it needs no
 * new page, or if all that it and the sequences before it ask for are no more
 * than the ring has; else it gets none. Pages are taken from the ring's
 * beginning in order of sequences; those behind what a sequence needs (ceil of
 * its slots, with the new rows, over page_size) go back behind the ring's end.
 * new_held and new_free_state (each may be the old one) receive the results,
 * offsets [batch + 1] the first row of each sequence, and for every row i <
 * rows sequences[i] (-1 behind the last), positions[i] (seen[b], or
 * lengths[b], + its place among the sequence's rows; 0) and slots[i]
 * (page * page_size + the slot in it; -1), each optional (NULL). Error bit 4: a
 * length, count or page count out of range (clamped), more slots than a row of
 * the table has (the sequence gets no rows), a page id out of range, more rows
 * than `rows` (dropped), a free_state out of range (no page moves). */
typedef struct fer_paged_plan_args {
    int32_t* page_table;         /* [batch, max_pages] */
    const int32_t* lengths;      /* [batch] */
    const int32_t* counts;       /* [batch] */
    const int32_t* held;         /* [batch] */
    const int32_t* seen;         /* [batch] or NULL: lengths */
    int32_t* free_pages;         /* [pages] */
    const int32_t* free_state;   /* [2] */
    int32_t* new_held;
    int32_t* new_free_state;
    int32_t* offsets;            /* [batch + 1] */
    int32_t* sequences;          /* [rows] or NULL, as the next two */
    int32_t* positions;
    int32_t* slots;
    int batch, max_pages, pages, page_size, rows;
} fer_paged_plan_args_t;
cudaError_t fer_paged_plan(const fer_paged_plan_args_t* args, uint32_t* err, cudaStream_t s);
/* Attention of rows of prompts or single tokens over the view's cache, keys
 * stored first: rows offsets[b] .. offsets[b+1] - 1 of q [rows, heads *
 * head_dim] are the last slots of sequence b < n_seq (offsets NULL: row b is
 * sequence b's last, and rows == n_seq). The row of slot p sees the slots s <= p
 * with s > p - window or s < sinks; window 0: all s <= p. Pages without a slot
 * that one of the call's rows sees are not read, nor are their entries. Other
 * arguments as fer_paged_attention's; lse [rows, heads]. A row that sees nothing
 * gives zeros, lse -inf; rows behind the last offset are left as they were.
 * Offsets that decrease or leave 0 .. rows set error bit 4, and out and lse are
 * then left as they were. The same bits run to run. workspace:
 * fer_paged_window_attention_workspace_bytes, rules as above; fewer rows may need
 * more bytes, so a buffer for calls of several sizes is as large as the largest of
 * their needs. The same holds for the prefix's workspace. */
typedef struct fer_paged_window_args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int rows, n_seq, heads;
    const int32_t* offsets;      /* [n_seq + 1] or NULL */
    int window, sinks;
    float scale;
    float* lse;
    void* workspace;
    size_t workspace_bytes;
} fer_paged_window_args_t;
size_t fer_paged_window_attention_workspace_bytes(int rows, int n_seq, int heads, int kv_heads, int head_dim,
                                                  int max_slots, int window, int sinks);
cudaError_t fer_paged_window_attention(const fer_paged_view_t* cache, const fer_paged_window_args_t* args, uint32_t* err,
                                       cudaStream_t s);
/* Attention of one query per sequence b < n_seq over the slots 0 ..
 * *prefix_length - 1 of prefix_pages, pages of the same pools that all sequences
 * share, and then the sequence's own held slots: one softmax over both. The
 * prefix is read once for all. A prefix_length out of range is clamped with
 * error bit 4. Other arguments as fer_paged_attention's. */
typedef struct fer_paged_prefix_args {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    int n_seq, heads;
    const int32_t* prefix_pages;   /* [max_prefix_pages] */
    const int32_t* prefix_length;  /* [1] */
    int max_prefix_pages;
    float scale;
    float* lse;
    void* workspace;
    size_t workspace_bytes;
} fer_paged_prefix_args_t;
size_t fer_paged_prefix_attention_workspace_bytes(int n_seq, int heads, int kv_heads, int head_dim, int max_slots,
                                                  int max_prefix_slots);
cudaError_t fer_paged_prefix_attention(const fer_paged_view_t* cache, const fer_paged_prefix_args_t* args, uint32_t* err,
                                       cudaStream_t s);
/* Per-token layer norm, x f32 [T, d] -> out bf16, d one of 128, 256, ..., 4096. */
cudaError_t fer_ln_bf16(const float* x, const float* g, const float* b, void* out, int T, int d, float eps,
                        cudaStream_t s);
/* x[t] = emb[tok[t]] as f32, emb bf16 [vocab, d], d % 256 == 0; an id outside
 * the vocabulary gives a zero row and error bit 4. */
cudaError_t fer_embed_f32(const int* tok, const void* emb, float* x, int T, int d, int vocab, uint32_t* err,
                          cudaStream_t s);
/* out[i] = bf16(stddev * N(0,1)), element i from draws 2i+1 and 2i+2 of the
 * splitmix64 stream of `seed` (Box-Muller). */
cudaError_t fer_fill_normal_bf16(void* out, size_t n, uint64_t seed, float stddev, cudaStream_t s);
cudaError_t fer_fill_f32(float* out, size_t n, float v, cudaStream_t s);
/* Fills `bytes` at dst (16-byte aligned) with the 32-bit pattern `value`
 * (trailing bytes short of a 16-byte word take its low byte). */
cudaError_t fer_fill_u32(void* dst, size_t bytes, uint32_t value, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FERCUDA_B200_NATIVE_H */
