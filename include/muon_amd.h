/*
 * muon_amd.h — C ABI of the MI355X-native Muon optimizer step (libmuon_amd.so).
 *
 * The library replaces the device-side work of muonium's `Muon.step()` hot path
 * (tonyf/dtensor-muon, package `muonium`). Every entry point takes plain device
 * pointers, sizes and a hipStream_t passed as `void*`; nothing allocates, frees or
 * synchronizes: the caller (the Python host package, or any FFI user) owns every
 * buffer. All launches are asynchronous on the given stream.
 *
 * Return value: MUON_OK (0) or one of the MUON_ERR_* codes; the text of the last
 * error on the calling thread is available from muon_amd_last_error().
 *
 * Shapes. A "tensor" handed to the step entry points is `nb` stored matrices of
 * `rows x cols`, contiguous (row-major, matrix after matrix): the transformed
 * gradient shape of muonium's `_init_muon_group` (optim.py:395-401). The
 * orthogonalization runs on the wide orientation X (m x n, m = min(rows, cols)),
 * transposing tall matrices as pe_loop/ns_loop do (polar_express.py:52-54,
 * newton_schulz.py:41-43).
 *
 * Workspace. The iteration works in a caller-allocated workspace whose size comes
 * from muon_orth_workspace_bytes(); the same (dtype, batch, rows, cols) quadruple
 * must be passed to every call that touches it. Its contents need no
 * initialization: every call rewrites what it reads later.
 */
#ifndef MUON_AMD_H
#define MUON_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* dtype codes */
#define MUON_DT_F32 0
#define MUON_DT_BF16 1
#define MUON_DT_F16 2

/* status codes */
#define MUON_OK 0
#define MUON_ERR_SHAPE 1
#define MUON_ERR_DTYPE 2
#define MUON_ERR_ALIGN 3
#define MUON_ERR_LAUNCH 4
#define MUON_ERR_ARG 5
#define MUON_ERR_DEVICE 6

/* quantized-state formats (muon_lp_*) */
#define MUON_Q_8BIT 8
#define MUON_Q_4BIT 4
#define MUON_Q_FP8 0

/* Maximum tensors per multi-tensor launch; larger lists are chunked internally. */
#define MUON_MAX_TENSORS 32

/* ABI version of this header (bumped on any signature change): 5. */
int muon_amd_abi_version(void);

/* Text of the last error reported on the calling thread ("" if none). */
const char* muon_amd_last_error(void);

/* Checks that the current HIP device is a gfx950 (MI355X) and that the code
 * objects load. No counterpart in the reference (Triton JIT-compiles on first use). */
int muon_amd_init(void);

/* ---- Gram kernel -------------------------------------------------------------
 * y[b] = x[b] @ x[b]^T for b < batch; x is (batch, M, K) contiguous, y is
 * (batch, M, M) contiguous, both `dtype` (bf16 or fp32), fp32 accumulation, output
 * exactly symmetric (upper-triangle tiles computed, lower mirrored).
 * Replaces: muonium/kernels/gram.py:109-152 `gram_(d_in, d_out)` (the Triton
 * `gram_nd`, gram.py:21-106). The contract checks of gram.py:114-130 live in the
 * Python wrapper, which raises the reference's AssertionError. */
int muon_gram(const void* x, void* y, int dtype, int64_t batch, int64_t M, int64_t K,
              void* stream);

/* ---- Orthogonalization workspace ---------------------------------------------- */
int64_t muon_orth_workspace_bytes(int dtype, int64_t batch, int64_t rows, int64_t cols);

/* Location of the orthogonalized result U (rows x cols) inside the workspace after
 * muon_orth_run(..., steps, ...): byte offset of matrix 0, row pitch and matrix stride
 * in elements of the wide iterate (m x n). *transposed is 1 for a tall matrix
 * (rows > cols), whose U(r, c) is then at row c, column r of that iterate. */
int muon_orth_result(int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
                     int64_t* offset_bytes, int64_t* row_pitch, int64_t* matrix_stride,
                     int* transposed);

/* ---- Pre-pass: momentum / Nesterov -> bf16 X (both layouts) + norm partials ------
 * For tensor t < ntensors (each nb matrices of rows x cols, elementwise):
 *   g  = maximize ? -grad : grad                                  (muon.py:41-42)
 *   buf' = buf * momentum + g        (fp32 math, stored in buf's dtype) (muon.py:49-50)
 *   g' = nesterov ? g + buf' * momentum : buf'                     (muon.py:53-56)
 *   X[t*nb + i] = cast(g', iteration dtype)                        (orthogonalize.py:101-102)
 * With bufs == NULL the momentum step is skipped (g' = g): the zeropower cast path.
 * write_back_grad stores g' into grad (the foreach driver's in-place Nesterov
 * update of the gradient list, muon.py:117-118). The sum of squares of the cast
 * values is accumulated per matrix for the Frobenius prescale (polar_express.py:89).
 * With ws == NULL only the momentum step runs (buf' in place, g' into grad when
 * write_back_grad): for a caller-supplied orthogonalizer that needs g' as a tensor.
 * Replaces: muonium/optim/algorithms/muon.py:39-56 and :108-119, plus the
 * `torch.stack(...).bfloat16()` of orthogonalize.py:159-161. */
int muon_prepass(int ntensors, void* const* grads, void* const* bufs, int g_dtype,
                 int buf_dtype, int64_t nb, int64_t rows, int64_t cols, float momentum,
                 int nesterov, int maximize, int write_back_grad, void* ws, int ws_dtype,
                 int64_t ws_batch, void* stream);

/* ---- Iteration: Newton-Schulz / Polar Express on the workspace -----------------
 * For the first `batch` matrices of the workspace: X /= (||X||_F * prescale + eps),
 * then for each of `steps` coefficient triples (a, b, c) (coeffs is steps*3 doubles):
 *   A = X X^T;  B = b*A + c*A A;  X = a*X + B X
 * in bf16 (fp32 accumulation) or fp32 according to ws_dtype.
 * Replaces: muonium/orthogonalize/polar_express.py:71-115 `pe_loop_triton`
 * (prescale 1.02) and newton_schulz.py:60-107 `ns_loop_triton` (prescale 1.0). */
int muon_orth_run(void* ws, int ws_dtype, int64_t ws_batch, int64_t batch, int64_t rows,
                  int64_t cols, const double* coeffs, int steps, float prescale, float eps,
                  void* stream);

/* muon_orth_run followed by muon_postpass of its result (u = NULL, the same arguments),
 * with the post-pass fused into the last iteration's X = a*X + B X where the shapes allow
 * (bf16 workspace; bf16 parameters, or fp32 / fp16 ones in launches small enough that the
 * fused form is the faster one; on the iterate's short side more than 64 rows, or at most 64
 * with bf16 parameters stored wide; ntensors * nb == batch, parameter rows a multiple of 8
 * elements in the stored orientation, 16-byte aligned parameters; the last product launches
 * once per 128 tensors): each bf16 element of the last X' is applied to its parameter element
 * (cautious weight decay and the shape-scaled step, exactly as muon_postpass) and X' is
 * not stored, so the workspace does not hold U afterwards. Otherwise the two calls run
 * one after the other. Replaces the orthogonalize-then-apply sequence of
 * muonium/optim/algorithms/muon.py:101-140 (foreach_update) and :58-77 (update). */
int muon_orth_run_apply(void* ws, int ws_dtype, int64_t ws_batch, int64_t batch, int64_t rows,
                        int64_t cols, const double* coeffs, int steps, float prescale,
                        float eps, int ntensors, void* const* params, int p_dtype, int64_t nb,
                        const float* adjusted_lrs, float wd, int cautious, void* stream);

/* muon_orth_run / muon_orth_run_apply for calls whose launches may run beside other calls'
 * launches on other streams (beside != 0): where two tile sizes of a product take about as
 * long, the one that leaves more of the device to the others. The results are bit for bit
 * the same. */
int muon_orth_run_beside(void* ws, int ws_dtype, int64_t ws_batch, int64_t batch, int64_t rows,
                         int64_t cols, const double* coeffs, int steps, float prescale, float eps,
                         int beside, void* stream);
int muon_orth_run_apply_beside(void* ws, int ws_dtype, int64_t ws_batch, int64_t batch,
                               int64_t rows, int64_t cols, const double* coeffs, int steps,
                               float prescale, float eps, int ntensors, void* const* params,
                               int p_dtype, int64_t nb, const float* adjusted_lrs, float wd,
                               int cautious, int beside, void* stream);

/* The iteration of several buckets (different extents, each with a bf16 workspace of its own whose
 * pre-pass has run) in common launches, and the apply of the buckets that name parameters
 * (ntensors > 0): bit for bit what one muon_orth_run (ntensors == 0, U stays in the workspace) or
 * muon_orth_run_apply per bucket gives. For buckets too small to fill the device: one launch
 * per product of an iteration instead of one per bucket. */
typedef struct MuonBucket {
  void* ws;
  int64_t ws_batch, batch, rows, cols;
  int ntensors, p_dtype;
  int64_t nb;
  void* const* params;
  const float* adjusted_lrs;
} MuonBucket;
int muon_orth_run_group(int nbuckets, const MuonBucket* buckets, const double* coeffs, int steps,
                        float prescale, float eps, float wd, int cautious, void* stream);

/* Copy U (first `batch` matrices, stored layout) out of the workspace into a
 * contiguous (batch, rows, cols) tensor of out_dtype. Replaces the return/unbind of
 * orthogonalize.py:101-102, :159-162. */
int muon_orth_extract(const void* ws, int ws_dtype, int64_t ws_batch, int64_t batch,
                      int64_t rows, int64_t cols, int steps, void* out, int out_dtype,
                      void* stream);

/* ---- Post-pass: cautious weight decay + shape-scaled apply ----------------------
 * For tensor t, element e (u from the workspace when u == NULL, else from the
 * contiguous tensor u of u_dtype holding ntensors*nb*rows*cols elements):
 *   v = wd != 0 ? (cautious ? u + (wd*p)*(u*p > 0) : u + wd*p) : u    (muon.py:62-69)
 *   p = round(p - adjusted_lrs[t] * v)                                 (muon.py:71-77)
 * in fp32 with no contraction; when wd == 0 the product adjusted_lr*u keeps u's dtype
 * (eager type promotion of a 0-dim fp32 tensor times a bf16 tensor: adjusted_lr is cast
 * to u's dtype, the product rounded to it). With u_scales (one per tensor, NULL for none)
 * u is first replaced by u * u_scales[t] rounded to u's dtype: the split_sizes row-block
 * rescale `u * scales[i]` of base.py:98 applied to a block handed over as its own tensor.
 * Replaces: muonium/optim/algorithms/muon.py:59-77 and :121-140. */
int muon_postpass(int ntensors, void* const* params, int p_dtype, const void* u, int u_dtype,
                  const void* ws, int ws_dtype, int64_t ws_batch, int steps, int64_t nb,
                  int64_t rows, int64_t cols, const float* adjusted_lrs, const float* u_scales,
                  float wd, int cautious, void* stream);

/* ---- NorMuon post-pass ------------------------------------------------------------
 * muon_postpass for the "normuon" algorithm: the update U (from the workspace when
 * u == NULL, else the contiguous tensor u of u_dtype, as in muon_postpass) is first
 * normalized per stored row (normuon.py:16-55), per row block when split_sizes is given
 * (nsplits blocks of stored rows summing to `rows`, at most MUON_MAX_SPLITS):
 *   r_i   = mean_j U(i, j)^2                          (fp32)
 *   v_i'  = lerp(v_i, r_i, 1 - beta2)                 (torch.lerp; v = variances[t], one
 *                                                      value per stored row, v_dtype)
 *   U'    = U(i, :) / (sqrt(v_i') + 1e-8)
 *   U''   = U' * ||U||_F / max(||U'||_F, 1e-8)        (norms per matrix and row block)
 * and v_i' is stored into the variance state; then cautious weight decay and the apply
 * run on U'' in fp32 exactly as muon_postpass. With u_scales (one per tensor, NULL for
 * none) U is first replaced by U * u_scales[t] rounded to U's dtype, before the statistics:
 * the split_sizes row-block rescale `u * scales[i]` of base.py:98, for a row block handed
 * over as its own tensor. The workspace (same quadruple as the other calls; required also
 * with an explicit u) holds the per-row scratch.
 * Replaces: muonium/optim/algorithms/normuon.py:16-55 (_normuon_normalize), :118-134
 * (NorMuon.update after the orthogonalization) and :182-203 (foreach_update). */
#define MUON_MAX_SPLITS 16
int muon_normuon_postpass(int ntensors, void* const* params, int p_dtype,
                          void* const* variances, int v_dtype, const void* u, int u_dtype,
                          void* ws, int ws_dtype, int64_t ws_batch, int steps, int64_t nb,
                          int64_t rows, int64_t cols, const int64_t* split_sizes, int nsplits,
                          const float* adjusted_lrs, const float* u_scales, float wd,
                          int cautious, double beta2, void* stream);

/* ---- Allocation-free NorMuon post-pass ------------------------------------------------
 * No counterpart in the reference: for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving or training loops, harnesses that forbid
 * hipMalloc). Same arithmetic and results as muon_normuon_postpass with an explicit update
 * u (required here) and no workspace: the per-row statistics live in a static device array
 * of MUON_NOALLOC_SCRATCH_BYTES per GPU, held until the process ends. A call needs
 * min(ntensors, MUON_MAX_TENSORS) * nb * rows * 4 bytes of it and is refused with
 * MUON_ERR_SHAPE beyond (rows up to 131072 for 32 single-matrix tensors). Nothing is
 * allocated and nothing needs clearing between calls (every value read is written first
 * by the same call). All calls on one GPU share its array: calls that overlap in time on
 * one GPU (on different streams) race and must be serialized by the caller. */
#define MUON_NOALLOC_SCRATCH_BYTES (16 * 1024 * 1024)
int muon_normuon_postpass_noalloc(int ntensors, void* const* params, int p_dtype,
                                  void* const* variances, int v_dtype, const void* u,
                                  int u_dtype, int64_t nb, int64_t rows, int64_t cols,
                                  const int64_t* split_sizes, int nsplits,
                                  const float* adjusted_lrs, const float* u_scales, float wd,
                                  int cautious, double beta2, void* stream);

/* ---- Quantized momentum (MuonLP) -------------------------------------------------
 * State of one tensor of `numel` values: codes (uint8; numel bytes for 8-bit and
 * fp8, numel/2 for 4-bit with element 2i in the high nibble) and one fp32 scale per
 * block of `block` consecutive values. 8/4-bit codes index the 256/16-entry fp32
 * `qmap`; value = qmap[code] * scale. fp8 codes are float8_e4m3fn; value =
 * float(code) * scale. Quantizing a block: absmax = max(|x|) clipped at 1e-12;
 * scale = absmax (fp8: absmax / 448); y = x / scale (IEEE division); 8/4-bit code =
 * largest i with qmap[i] <= y, then i+1 if y - qmap[i] >= (qmap[i+1]-qmap[i])*0.5.
 * Replaces the torchao 0.17.0 OptimState8bit / OptimState4bit / OptimStateFp8
 * arithmetic reached from muonium/optim/optim_lp.py:118-133 via muon.py:45,50. */
int muon_lp_quantize(const float* src, void* codes, float* scales, const float* qmap,
                     int qformat, int64_t numel, int64_t block, void* stream);
int muon_lp_dequantize(const void* codes, const float* scales, const float* qmap,
                       int qformat, int64_t numel, int64_t block, float* dst, void* stream);

/* Fused dequant -> momentum -> requant pre-pass for quantized momentum buffers:
 * as muon_prepass, with buf = dequant(codes, scales) and buf' requantized in
 * place; Nesterov uses the unquantized buf' (muon.py:49-56). */
int muon_lp_prepass(int ntensors, void* const* grads, int g_dtype, void* const* codes,
                    void* const* scales, const float* qmap, int qformat, int64_t block,
                    int64_t nb, int64_t rows, int64_t cols, float momentum, int nesterov,
                    int maximize, void* ws, int ws_dtype, int64_t ws_batch, void* stream);

/* ---- Row operators of the training step -----------------------------------------------
 * No counterpart in the reference: what a model's forward and backward pass computes beside
 * its matrix products and attention, where this optimizer's parameters are trained. Inputs of
 * fp32, bf16 or fp16, every sum and exponential in fp32 or more, one rounding at the output.
 * Strides are in elements; the last dimension is contiguous. Nothing is allocated; a call is
 * one to three launches on the given stream, with the same bits on every run.
 *
 * Queries and keys: per head of `dim` values (at most 1024) the RMS norm
 * n = x / sqrt(mean(x^2) + eps) * weight, and the rotation of its first `rotary` values (even)
 * by the angles of the token's position: (a c - b s, b c + a s) for the pairs (i, i + rotary/2),
 * or (2i, 2i+1) when interleaved. strides: batch, token, head of q, then of k (backward: then of
 * dq_out and dk_out); outputs and dq, dk are contiguous (batch, tokens, heads, dim). Weights
 * (w_dtype, dim values) may be NULL. cos and sin are (table_len, rotary/2) fp32; positions
 * (pos_bits 32 or 64; NULL: token t is at t) may be shared by the batches
 * (pos_batch_stride 0). A position outside the table gives NaN, and nothing is read there.
 * The backward pass needs ws of muon_qk_norm_rope_workspace_bytes(dim) for weight gradients. */
int muon_qk_norm_rope(const void* q, const void* k, const int64_t* strides, const void* q_weight,
                      const void* k_weight, int w_dtype, const float* cosv, const float* sinv,
                      int64_t table_len, const void* positions, int pos_bits,
                      int64_t pos_batch_stride, void* q_out, void* k_out, int dtype, int64_t batch,
                      int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim,
                      int64_t rotary, int interleaved, float eps, void* stream);
int64_t muon_qk_norm_rope_workspace_bytes(int64_t dim);
int muon_qk_norm_rope_backward(const void* q, const void* k, const void* dq_out,
                               const void* dk_out, const int64_t* strides, const void* q_weight,
                               const void* k_weight, int w_dtype, const float* cosv,
                               const float* sinv, int64_t table_len, const void* positions,
                               int pos_bits, int64_t pos_batch_stride, void* dq, void* dk,
                               void* dq_weight, void* dk_weight, void* ws, int dtype,
                               int64_t batch, int64_t tokens, int64_t q_heads, int64_t k_heads,
                               int64_t dim, int64_t rotary, int interleaved, float eps,
                               void* stream);

/* Expert routing of (tokens, experts) logits (at most 1024 experts): the `top` (at most 64)
 * largest logits of each token in descending order, ties by the lower index, a NaN as the
 * largest; an expert at -inf is never chosen, and a slot that finds none holds -1 with gate 0.
 * gates (tokens, top) fp32: the softmax values, or (normalize) these over their sum. Tokens
 * whose token_mask byte is 0 (NULL: none) and tokens with all logits -inf choose nothing and
 * count nowhere. Over the N others (*kept): counts[e] = tokens that chose e;
 * balance = experts * sum_e counts[e] / (top N) * mean_t softmax_te; zloss = mean_t lse_t^2
 * (both 0 for N = 0). Any of dgates, dbalance, dzloss may be NULL (no gradient from there). */
int64_t muon_route_workspace_bytes(int64_t tokens, int64_t experts);
int muon_route(const void* logits, int dtype, int64_t row_stride, int64_t tokens, int64_t experts,
               int64_t top, int normalize, const void* token_mask, float* gates,
               int64_t* chosen, int64_t* counts, float* balance, float* zloss, float* kept,
               void* ws, void* stream);
int muon_route_backward(const void* logits, int dtype, int64_t row_stride, int64_t tokens,
                        int64_t experts, int64_t top, int normalize, const void* token_mask,
                        const int64_t* chosen, const int64_t* counts, const float* kept,
                        const float* dgates, const float* dbalance, const float* dzloss,
                        void* dlogits, void* stream);

/* logprobs[n] = log softmax(logits[n] / temperature)[tokens[n]] in fp32. A negative token leaves
 * its row out (0, and no gradient; the row is not read); one of `vocab` or more gives NaN. stats
 * (2 * rows floats, NULL: not kept) is what the backward pass needs beside the logits, ws holds
 * muon_token_logprobs_workspace_bytes (0: may be NULL). Backward: dlogits (rows, vocab), contiguous, from
 * dlogprobs (rows) times *scale (NULL: 1); a row whose gradient is 0 is not read, and gets 0
 * whatever *scale is. */
int64_t muon_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab);
int muon_token_logprobs(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                        int64_t vocab, const int64_t* tokens, float temperature, float* logprobs,
                        float* stats, void* ws, void* stream);
int muon_token_logprobs_backward(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                                 int64_t vocab, const int64_t* tokens, float temperature,
                                 const float* stats, const float* dlogprobs, const float* scale,
                                 void* dlogits, void* stream);

/* The clipped policy loss: with r = exp(logprob - old), per row
 *   term = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
 *          + kl_coef (exp(ref - logprob) - (ref - logprob) - 1)      (ref_logprobs NULL: without)
 * and *loss = sum weights * term. Rows of weight 0 are left out like negative tokens. terms holds
 * one float a row. The gradient either in the same pass (dlogits, for a loss gradient of 1; where
 * muon_policy_loss_one_pass says the row fits a workgroup's registers), or later by
 * muon_token_logprobs_backward with dlogprobs = coef and the kept stats (both may be NULL
 * when not needed). muon_policy_loss_rescale takes the dlogits of the same pass, with the coef
 * and stats that it kept, to the loss gradient *scale: it makes the rows that have a gradient again
 * from the logits, each value rounded once (a scale of 1 touches nothing).
 * muon_scale_gradient multiplies any n values by *scale in place, the rounded ones (a
 * scale of 1 touches nothing). */
int muon_policy_loss_one_pass(int dtype, int64_t vocab);
int muon_policy_loss(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                     int64_t vocab, const int64_t* tokens, const float* old_logprobs,
                     const float* advantages, const float* weights, const float* ref_logprobs,
                     float clip_low, float clip_high, float kl_coef, float temperature,
                     float* loss, float* logprobs, float* terms, float* stats, float* coef,
                     void* dlogits, void* ws, void* stream);
int muon_policy_loss_rescale(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                             int64_t vocab, const int64_t* tokens, float temperature,
                             const float* stats, const float* coef, const float* scale,
                             void* dlogits, void* stream);
int muon_scale_gradient(void* x, int dtype, int64_t n, const float* scale, void* stream);

/* ---- Experts: routed tokens to their experts and back -------------------------------------
 * No counterpart in the reference: what carries out the choices of muon_route.
 *
 * muon_expert_order: the rows of all choices (tokens x top, below 2^31) sorted by expert (at most
 * 1024), in the order of choices within one: slots[i] = choice i's row; a choice whose number is none
 * of 0 .. nexperts - 1 is empty, comes behind the last expert's, and has slots[i] = -1 - its row.
 * offsets (nexperts + 1): the experts' first rows, and the end of the last one's.
 * muon_dispatch: rows (tokens * top, width), contiguous, rows[slot] = x[token]; an empty choice's row
 * is 0. muon_combine: y (tokens, width), contiguous, y[t] = sum_j gates[t, j] rows[slot(t, j)] over the
 * kept choices (gates NULL: ones, the gradient of muon_dispatch). muon_combine_backward: drows like
 * muon_dispatch's rows, gates[t, j] dy[t], and dgates[t, j] = <dy[t], rows[slot]>; either may be NULL.
 * Gates and rows of empty choices reach nothing, their gradients are 0. A slot outside the rows is
 * left out. Strides of rows in elements, columns contiguous; sums in fp32, rounded once. */
int64_t muon_expert_order_workspace_bytes(int64_t choices, int64_t nexperts);
int muon_expert_order(const int64_t* experts, int64_t choices, int64_t nexperts, int32_t* slots,
                      int32_t* offsets, void* ws, void* stream);
int muon_dispatch(const void* x, int dtype, int64_t row_stride, int64_t tokens, int64_t top,
                  int64_t width, const int32_t* slots, void* rows, void* stream);
int muon_combine(const void* rows, int dtype, int64_t row_stride, int64_t tokens, int64_t top,
                 int64_t width, const int32_t* slots, const float* gates, void* y, void* stream);
int muon_combine_backward(const void* dy, int64_t dy_stride, const void* rows, int64_t row_stride,
                          int dtype, int64_t tokens, int64_t top, int64_t width,
                          const int32_t* slots, const float* gates, void* drows, float* dgates,
                          void* stream);

/* The experts' matrices, weight (experts, out, in), contiguous, on their rows offsets[e] ..
 * offsets[e + 1] - 1 of `nrows`: y = x W_e^T (nrows, out); drows = dy W_e (nrows, in); dweight_e =
 * dy_e^T x_e (experts, out, in), 0 for an expert without rows; all contiguous. Rows behind
 * offsets[experts] give zeros and reach nothing. Products of 16-bit types on the matrix cores with
 * fp32 sums; fp32 in fp32. offsets[0] counts as 0, and the others, which have to rise, are taken
 * into 0 .. nrows: nothing is read out of range whatever they hold. */
int muon_expert_linear(const void* rows, int dtype, int64_t row_stride, int64_t nrows,
                       int64_t experts, int64_t out, int64_t in, const void* weight,
                       const int32_t* offsets, void* y, void* stream);
int muon_expert_linear_backward_rows(const void* dy, int dtype, int64_t dy_stride, int64_t nrows,
                                     int64_t experts, int64_t out, int64_t in, const void* weight,
                                     const int32_t* offsets, void* drows, void* stream);
int muon_expert_linear_backward_weight(const void* dy, int dtype, int64_t dy_stride,
                                       const void* rows, int64_t row_stride, int64_t nrows,
                                       int64_t experts, int64_t out, int64_t in,
                                       const int32_t* offsets, void* dweight, void* stream);

/* ---- AdamW over many tensors -------------------------------------------------------------
 * One step of every tensor, in place: with t = ++*step (fp32, on the device),
 *   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
 *   p = (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 * (maximize: with -g), in fp32, p rounded once. Parameters and gradients are of one type and order of
 * values. block 0: exp_avg and exp_avg_sq are fp32 m and v, the scales unused. block a power of two from
 * 64 to 2048 that divides numel: they are float8_e4m3fn codes of m and of sqrt(v), value = float(code) *
 * scale of its block, scale = max(absmax, 1e-12) / 448. Codes are the nearest ones, to even, or, from beta1 =
 * 0.9375 on or above beta2 = 0.95, where the nearest would keep moments where they are, one of the two around
 * the value at random (by step and place: the same ones every time); a root's code is the least one, 1, in
 * place of 0 where the mean's is not 0, and with the nearest codes a mean below 8 of them whose gradient is 0
 * gives up half of one beside its decay. No two tensors may share memory. ws:
 * muon_adamw_workspace_bytes. `tensors` is host memory, read before the call returns. */
typedef struct MuonAdamTensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* avg_scale;
  float* sq_scale;
  float* step;
  int64_t numel;
} MuonAdamTensor;
int64_t muon_adamw_workspace_bytes(int64_t ntensors);
int muon_adamw(int64_t ntensors, const MuonAdamTensor* tensors, int dtype, int64_t block, double lr,
               double beta1, double beta2, double eps, double weight_decay, int maximize, void* ws,
               void* stream);

/* ---- Kernel timing (measurement support) ------------------------------------------
 * No counterpart in the reference. While enabled, every kernel the step entry points
 * launch is bracketed by hipEvents on its own stream; muon_timing_read() waits for
 * the last event and returns, per kernel kind (MUON_K_*), the summed duration in ms,
 * the launch count and the summed algorithmic work (FLOP for the products, bytes for
 * the elementwise passes, as documented per kind). Capacity: 65536 launches. */
#define MUON_K_SYRK_XX 0   /* A = X X^T: m(m+1) n FLOP per matrix (upper triangle) */
#define MUON_K_SYRK_AA 1   /* B = b A + c A A: m(m+1) m FLOP per matrix */
#define MUON_K_GEMM_BX 2   /* X = a X + B X: 2 m^2 n FLOP per matrix */
#define MUON_K_PREPASS 3   /* bytes: grad + 2 * buffer + one bf16 X per element */
#define MUON_K_POSTPASS 4  /* bytes: u + 2 * param per element */
#define MUON_K_LP_PREPASS 5 /* bytes: grad + 2 * codes + 2 * scales + one bf16 X */
#define MUON_K_OTHER 6     /* finalize / transpose / scale / extract (no work counted) */
#define MUON_K_GEMM_BX_APPLY 7 /* the last X = a X + B X with the post-pass fused
                                  (muon_orth_run_apply): 2 m^2 n FLOP per matrix; the apply
                                  moves 2 * param bytes per element besides */
#define MUON_K_COUNT 8
int muon_timing_enable(int on);
int muon_timing_read(double* ms, int64_t* launches, double* work);

#ifdef __cplusplus
}
#endif

#endif /* MUON_AMD_H */
