/*
 * trnfft_amd.h — C ABI of the MI355X (gfx950) FFT backend for trnfft.
 *
 * Plain C: raw device pointers, sizes and an opaque stream handle; no torch types.  Data is in
 * trnfft's split layout (ComplexTensor, trnfft/complex.py:16-33): two contiguous row-major
 * fp32 planes, re and im, batch rows of length n.  All entry points return TFA_OK (0) or a
 * negative status; tfa_last_error() gives the calling thread's message for the last failure.
 *
 * Ownership: the caller owns every input, output and workspace buffer (device memory, e.g. from
 * the PyTorch caching allocator).  A plan owns its device tables (twiddles, Bluestein chirp and
 * filter spectrum, DFT matrix) and is immutable after creation, so tfa_execute* may be called
 * concurrently on one plan from several threads/streams.  A plan is bound to the device that was
 * current at creation.
 */
#ifndef TRNFFT_AMD_H
#define TRNFFT_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct tfa_plan tfa_plan;
typedef void* tfa_stream; /* hipStream_t; NULL = the null stream */

/* Status codes (the Python layer maps them to exceptions). */
#define TFA_OK 0
#define TFA_ERR_INVALID (-1)     /* bad argument                      -> ValueError          */
#define TFA_ERR_UNSUPPORTED (-2) /* size or kind not implemented      -> NotImplementedError */
#define TFA_ERR_HIP (-3)         /* HIP runtime / launch failure      -> RuntimeError        */

/* Plan kinds. */
#define TFA_KIND_C2C 0       /* power-of-two n (Stockham in LDS; four-step above 16384)     */
#define TFA_KIND_BLUESTEIN 1 /* any n >= 2, chirp-z over a power-of-two m >= 2n-1            */
#define TFA_KIND_DFT_GEMM 2  /* n <= 256, X = x @ W on the matrix cores                      */
#define TFA_KIND_STFT 3      /* framed, windowed onesided/twosided transform of real signals */
#define TFA_KIND_FFT2 4      /* 2-D transform over the last two axes (n = last, n2 = second to last) */
#define TFA_KIND_REAL 5      /* real rows: forward r2c (n real -> n/2+1 bins), inverse c2r; power-of-two 4 <= n <= 32768 */

/* STFT flags. */
#define TFA_STFT_CENTER 1     /* reflect-pad n_fft/2 on both sides (pad_mode="reflect") */
#define TFA_STFT_NORMALIZED 2 /* scale by 1/sqrt(n_fft)                                 */
#define TFA_STFT_ONESIDED 4   /* keep bins 0..n_fft/2                                   */
/* Spectra stored (batch, n_frames, n_bins) row-major instead of (batch, n_bins, n_frames).  Without
 * it the planes are trnfft's result layout: its stft wraps the transposed frame spectra in a
 * ComplexTensor, whose constructor makes them contiguous (trnfft/api.py:357-365,
 * trnfft/complex.py:29-33).  With it they are in the memory order of torch.stft's
 * (..., freq, time) result (no reference counterpart).  Applies to the forward output, the
 * inverse input and the backward's gradient input. */
#define TFA_STFT_FRAMES_MAJOR 8

typedef struct tfa_plan_desc {
  int32_t kind;    /* TFA_KIND_* */
  int32_t inverse; /* 0: forward, sign -1, unscaled; 1: inverse, sign +1, scaled 1/n */
  int64_t n;       /* transform length (STFT: n_fft) */
  int64_t hop;     /* STFT only: hop_length */
  int32_t flags;   /* STFT only: TFA_STFT_* */
  int32_t reserved;
  int64_t n2;      /* FFT2 only: length of the second-to-last axis */
} tfa_plan_desc;

/*
 * Create a plan.  Replaces the reference's per-call plan lookup plus table construction:
 * trnfft/plan.py:34-46 (create_plan: algorithm choice, Bluestein m = 1 << (2n-2).bit_length()),
 * trnfft/fft_core.py:86-88 (radix-2 twiddles), :1316-1345 (Bluestein chirp, with the same
 * fp32 angle expression sign*pi*k*k/n, and filter h), :239-243 (DFT matrix).
 */
int tfa_plan_create(tfa_plan** out, const tfa_plan_desc* desc);

/* Release a plan and its device tables (trnfft/plan.py:49-50 clear_plan_cache drops them). */
void tfa_plan_destroy(tfa_plan* plan);

/* Device workspace (bytes) tfa_execute needs for `batch` rows; 0 when none. */
int tfa_plan_workspace_size(const tfa_plan* plan, int64_t batch, size_t* bytes);

/* Padded length m of a Bluestein plan (n for the other kinds). */
int64_t tfa_plan_padded_n(const tfa_plan* plan);

/*
 * Batched 1-D transform along the last axis: out[b, k] = sum_j in[b, j] W^(j k) (x 1/n when
 * inverse).  in_im may be NULL for real input (imaginary part zero, trnfft/complex.py:27-28).
 * Out-of-place, or in place with out_* == in_*.  Replaces trnfft/fft_core.py:22-50 (fft_core),
 * which dispatches to _cooley_tukey (:53-117, power-of-two n), _bluestein (:1285-1376, other n)
 * and, for TFA_KIND_DFT_GEMM plans, _fft_via_gemm (:221-251).
 * TFA_KIND_FFT2 plans: `batch` arrays of (n2, n) each, transformed over both axes (x 1/(n n2)
 * when inverse), power-of-two 16 <= n <= 4096 and 16 <= n2 <= 4096 (two HBM passes), or
 * n * n2 <= 16384 with both axes >= 4 (>= 8 at 8192, >= 16 at 16384; whole images in LDS, one
 * pass); output must not alias the input; replaces trnfft/api.py:105-139 (fft2 -> fftn over
 * (-2, -1)).
 * TFA_KIND_REAL plans, forward (replaces trnfft/api.py:38-46, rfft): in_re = (batch, n) real
 * rows, in_im must be NULL, out_re/out_im = (batch, n/2+1) bins.  Inverse (replaces
 * trnfft/api.py:49-68, irfft with its default n = 2*(bins-1)): in_re/in_im = (batch, n/2+1)
 * bins, out_re = (batch, n) real rows scaled 1/n, out_im unused (may be NULL); the imaginary
 * parts of bins 0 and n/2 are ignored, as the reference's real part of the Hermitian-completed
 * inverse ignores them.  The real rows (input of the forward, output of the inverse) must be
 * 8-byte aligned; out-of-place only.
 */
int tfa_execute(const tfa_plan* plan, int64_t batch, const float* in_re, const float* in_im,
                float* out_re, float* out_im, void* workspace, tfa_stream stream);

/*
 * tfa_execute without a workspace argument and without any device allocation: the scratch the
 * four-step (n > 16384) and split-Bluestein kernels need comes from a static device array of
 * 64 MiB per GPU, part of the library's code object and held until the process ends.  No
 * counterpart in the reference; it is for callers that cannot allocate device memory (code under
 * HIP-graph capture, serving loops, harnesses that forbid hipMalloc).  A call whose scratch
 * (tfa_plan_workspace_size) exceeds 64 MiB fails with TFA_ERR_INVALID; plans that need no scratch
 * run exactly as tfa_execute.  Every call on one GPU shares that GPU's scratch: eager calls are
 * ordered on the device by the library (each waits, on its stream, for an event the previous
 * eager call recorded), but calls made while the stream is capturing a HIP graph are not, so
 * graph replays that overlap other noalloc calls on the same GPU race.
 */
int tfa_execute_noalloc(const tfa_plan* plan, int64_t batch, const float* in_re, const float* in_im,
                        float* out_re, float* out_im, tfa_stream stream);

/*
 * Batched 1-D transform along a strided axis, in place allowed: data viewed as (outer, n, stride)
 * row-major, each of the outer*stride columns transformed along its n elements (element stride
 * `stride`).  TFA_KIND_C2C plans with n <= 4096, or TFA_KIND_BLUESTEIN plans with n <= 2048
 * (padded length m <= 4096).  Replaces the transpose-copy + contiguous FFT + transpose-back of
 * trnfft/api.py:496-516 (_fft_along_dim) used by fft2/fftn/ifftn.
 */
int tfa_execute_strided(const tfa_plan* plan, int64_t outer, int64_t stride, const float* in_re,
                        const float* in_im, float* out_re, float* out_im, tfa_stream stream);

/*
 * tfa_execute_strided extended to power-of-two TFA_KIND_C2C axes 4096 < n <= 2^24 with
 * stride >= 4 (>= 8 from n = 2^21): two strided passes (three from 2^21) through `workspace`,
 * whose size tfa_strided_workspace_size reports (2 * 4 * outer * n * stride bytes for such axes,
 * else 0).  n = 4096 with stride >= 16 also takes two passes (faster than the single pass there).
 * In place allowed (out_* == in_*); the workspace must not overlap the data.  Every other
 * plan/stride goes to tfa_execute_strided (workspace unused).  outer = 0 is a no-op on both entry
 * points (the size query then reports 0 bytes).  Replaces the same transposes of
 * trnfft/api.py:496-516 for long axes.
 */
int tfa_strided_workspace_size(const tfa_plan* plan, int64_t outer, int64_t stride, size_t* bytes);
int tfa_execute_strided_ws(const tfa_plan* plan, int64_t outer, int64_t stride, const float* in_re,
                           const float* in_im, float* out_re, float* out_im, void* workspace, tfa_stream stream);

/*
 * Short-time Fourier transform of `batch` real signals of `num_samples` samples each.  Frames
 * of n_fft samples every hop, after reflect padding when TFA_STFT_CENTER; each frame is
 * multiplied by window (device pointer, n_fft floats, already centre-padded to n_fft) and
 * transformed; output planes are (batch, n_bins, n_frames) row-major, or (batch, n_frames,
 * n_bins) with TFA_STFT_FRAMES_MAJOR, with n_bins = n_fft/2+1 when TFA_STFT_ONESIDED else n_fft.  Replaces trnfft/api.py:291-365 (stft).  n_fft: a power
 * of two in [16, 4096], or any other n_fft from 9 up to 2731 (onesided) or 2048 (two-sided),
 * forward only: each frame then goes through the reference's Bluestein chain
 * (trnfft/fft_core.py:1285-1376), convolved at the shortest power of two or 3 * 2^k that holds
 * n_fft + n_bins - 1 points.
 */
int tfa_stft_frames(const tfa_plan* plan, int64_t num_samples, int64_t* n_frames);
int tfa_stft_execute(const tfa_plan* plan, int64_t batch, int64_t num_samples, const float* signal,
                     const float* window, float* out_re, float* out_im, tfa_stream stream);

/*
 * Complex GEMM on split planes, C = A @ B (b_trans = 0) or C = A @ B^T (b_trans = 1), plus an
 * optional complex bias broadcast over rows (bias_re/bias_im NULL for none).  A is (m, k) with
 * row stride lda; B is (k, n) with row stride ldb, or (n, k) when b_trans; C is (m, n) with row
 * stride ldc.  Replaces trnfft/nki/dispatch.py:74-84 (complex_gemm) and :91-102
 * (complex_linear: y = x @ W^T with W (out, in)), whose kernels are :121-200 and :267-345, and
 * the bias add of trnfft/nn.py:46-48.
 */
int tfa_complex_gemm(int64_t m, int64_t n, int64_t k, const float* a_re, const float* a_im,
                     int64_t lda, const float* b_re, const float* b_im, int64_t ldb, int32_t b_trans,
                     const float* bias_re, const float* bias_im, float* c_re, float* c_im,
                     int64_t ldc, tfa_stream stream);

/*
 * Inverse STFT (TFA_KIND_STFT plan created with inverse = 1; n = n_fft, hop, flags CENTER /
 * NORMALIZED / ONESIDED, FRAMES_MAJOR optional): spec_re/spec_im (batch, n_bins, n_frames), or
 * (batch, n_frames, n_bins) with FRAMES_MAJOR, with n_bins = n/2+1 when ONESIDED else n, -> out
 * (batch, out_len), out_len from tfa_istft_length (length < 0: the default length).
 * Hermitian completion (onesided) or the real part of each frame's inverse transform (two-sided,
 * power-of-two n only), inverse transform, window, overlap-add, division by the window-square
 * envelope where it exceeds 1e-8 (the raw overlap-add elsewhere), centre trim and zero fill to
 * `length` in one kernel.  Replaces trnfft/api.py:368-470 (istft), whose per-frame loops
 * (:438-452) and window-sum masking (:450-452) it fuses.
 */
int tfa_istft_length(const tfa_plan* plan, int64_t n_frames, int64_t length, int64_t* out_len);
int tfa_istft_execute(const tfa_plan* plan, int64_t batch, int64_t n_frames, const float* spec_re,
                      const float* spec_im, const float* window, float* out, int64_t length, tfa_stream stream);

/*
 * Gradient of the onesided forward STFT with respect to its padded signal: grad_re/grad_im
 * (batch, n/2+1, n_frames), or (batch, n_frames, n/2+1) when the plan has FRAMES_MAJOR, the
 * gradient of tfa_stft_execute's output planes, -> grad_padded
 * (batch, padded_len), padded_len = num_samples + 2*(n/2) when CENTER else num_samples, n_frames
 * = 1 + (padded_len - n)/hop.  Per frame the adjoint of the r2c transform (interior bins halved,
 * Hermitian-completed inverse transform, unscaled; 1/sqrt(n) when NORMALIZED), times the window,
 * overlap-added; samples no frame covers get zero.  n_fft that is not a power of two: per frame
 * the adjoint of the Bluestein chain the forward kernel runs (conj(chirp) times the gradient,
 * convolved with chirp[|s|], times conj(chirp)).  Undoing the centre padding (the reflected edges
 * folded back) is left to the caller.  Runs on the forward STFT plan of the call being
 * differentiated (ONESIDED required); a hop whose recomputed halo frames would fill the kernel's
 * frame tile returns TFA_ERR_UNSUPPORTED.  Replaces the backward that torch autograd derives for
 * trnfft/api.py:310-349 (pad, frame index, window multiply, per-frame transform): a
 * gather-transpose of the gradient, an inverse transform per frame and an index_add/fold
 * overlap-add.
 */
int tfa_stft_backward_execute(const tfa_plan* plan, int64_t batch, int64_t n_frames, const float* grad_re,
                              const float* grad_im, const float* window, float* grad_padded, int64_t padded_len,
                              tfa_stream stream);

/*
 * Rows around a complex transform of real data of any length (trnfft/api.py:38-68): with complete = 0 the first
 * `half` bins of (batch, n) rows, with complete = 1 the Hermitian rows of length n (half <= n <= 2 half - 1) of
 * (batch, half) bins, X_k = conj X_{n-k} for k >= half.  Out of place.
 */
int tfa_half_rows(int32_t complete, int64_t batch, int64_t n, int64_t half, const float* in_re, const float* in_im,
                  float* out_re, float* out_im, tfa_stream stream);

/*
 * The reflect padding's adjoint, in place on (batch, pad + length + pad) rows: each kept sample receives the
 * gradient of its mirror images, so that columns [pad, pad + length) are the gradient of the signal
 * (the backward of trnfft/api.py:310-313's F.pad).
 */
int tfa_stft_fold_edges(int64_t batch, int64_t pad, int64_t length, float* grad_padded, tfa_stream stream);

/* Operand ops of tfa_complex_gemm_ex (BLAS-style, plus conjugation without transpose). */
#define TFA_OP_N 0 /* op(X) = X          */
#define TFA_OP_T 1 /* op(X) = X^T        */
#define TFA_OP_C 2 /* op(X) = conj(X)^T  */
#define TFA_OP_R 3 /* op(X) = conj(X)    */

/*
 * General complex GEMM on split planes: C = alpha * op(A) @ op(B) + bias, op(A) (m, k), op(B)
 * (k, n).  A is stored (m, k), or (k, m) for TFA_OP_T/TFA_OP_C, with row stride lda; B is stored
 * (k, n), or (n, k) for TFA_OP_T/TFA_OP_C, with row stride ldb.  These are the adjoint products
 * of trnfft/nki/autograd.py:92-155 (_ComplexGEMMFn.backward dA = dC B^H, dB = A^H dC;
 * _ComplexLinearFn.backward dX = dY conj(W), dW = dY^T conj(X)), which the reference runs as
 * eight real torch matmuls; here each is one launch.
 */
int tfa_complex_gemm_ex(int64_t m, int64_t n, int64_t k, const float* a_re, const float* a_im, int64_t lda,
                        int32_t a_op, const float* b_re, const float* b_im, int64_t ldb, int32_t b_op, float alpha,
                        const float* bias_re, const float* bias_im, float* c_re, float* c_im, int64_t ldc,
                        tfa_stream stream);

/*
 * Strided-batched form of tfa_complex_gemm_ex: for b in [0, batch),
 *   C_b = alpha * op(A_b) @ op(B_b) + bias,  X_b = X + b * stride_x (floats, both planes).
 * A stride of 0 shares that operand across the batch (broadcast); C's stride must separate the
 * output matrices.  Replaces the batched and broadcast torch.matmul products of
 * trnfft/complex.py:142-150 (complex_matmul / ComplexTensor.__matmul__: four real matmuls of
 * (..., m, k) @ (..., k, n) operands), one launch for all four products of every matrix pair.
 */
int tfa_complex_gemm_batched(int64_t batch, int64_t m, int64_t n, int64_t k, const float* a_re, const float* a_im,
                             int64_t lda, int64_t stride_a, int32_t a_op, const float* b_re, const float* b_im,
                             int64_t ldb, int64_t stride_b, int32_t b_op, float alpha, const float* bias_re,
                             const float* bias_im, float* c_re, float* c_im, int64_t ldc, int64_t stride_c,
                             tfa_stream stream);

/*
 * tfa_complex_gemm_batched with scratch memory: a product of few output tiles and a long k (a
 * weight gradient) is summed over several k ranges at once, whose partial results `workspace`
 * (device memory of tfa_complex_gemm_workspace_size bytes, 0 for every other product; NULL: no
 * split) holds until a second launch adds them in a fixed order.
 */
int tfa_complex_gemm_workspace_size(int64_t batch, int64_t m, int64_t n, int64_t k, size_t* bytes);
int tfa_complex_gemm_ws(int64_t batch, int64_t m, int64_t n, int64_t k, const float* a_re, const float* a_im,
                        int64_t lda, int64_t stride_a, int32_t a_op, const float* b_re, const float* b_im, int64_t ldb,
                        int64_t stride_b, int32_t b_op, float alpha, const float* bias_re, const float* bias_im,
                        float* c_re, float* c_im, int64_t ldc, int64_t stride_c, void* workspace, tfa_stream stream);

/*
 * Sums over the rows of two row-major (rows, cols) planes (the bias gradient of
 * trnfft/nki/autograd.py:125-155).  `workspace`: tfa_column_sums_workspace_size bytes of device memory (NULL: the rows
 * are summed by one workgroup per 64 columns).
 */
int tfa_column_sums_workspace_size(int64_t rows, int64_t cols, size_t* bytes);
int tfa_column_sums(int64_t rows, int64_t cols, const float* re, const float* im, float* out_re, float* out_im,
                    void* workspace, tfa_stream stream);

/* ---- Operators of models on frames (no counterpart in the reference) ---------------------------------------------
 *
 * What a model that is trained on STFT frames needs next to the transforms and the complex products: a mixing over
 * frames with memory, a normalisation of channels-last features, and the optimizer's step.  Element types: */
#define TFA_DTYPE_F32 0
#define TFA_DTYPE_BF16 1
#define TFA_DTYPE_F16 2

/*
 * Linear attention with a decay for each head, over (batch, tokens, heads, features) operands:
 *   S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,   out_t = scale S_t^T q_t
 * q, k (key_dim features) and v (value_dim) may have fewer heads than the call: head h reads head h / (heads / own).
 * Their strides are in elements, for batch, token and head; features are contiguous and q, k, v, grad_out 16-byte aligned
 * (a step's operands may lie anywhere; operands whose features or strides are not multiples of 16 bytes are copied to the
 * workspace first).  State tensors are fp32 (batch, heads, key_dim, value_dim), the outputs contiguous (batch, tokens,
 * heads, value_dim).  log_decay: (heads) device fp32, at most 0 (-inf: no memory; above 0 the state grows).  lengths: (batch)
 * device int64 or NULL; tokens at and past a sequence's length are padding: never read, zero in the outputs and gradients,
 * and the state is the one at the length.  Products of bf16 operands are exact; scores, states and sums are held in fp32
 * for every type, and up to 128 features enter the products of 16-bit outputs with 16 to 17 bits.  What is not finite makes
 * NaN or infinities of what depends on it by the recurrence: its token and later ones.  Head dimensions up to 256.
 */
typedef struct tfa_attn_desc {
  int32_t dtype; /* TFA_DTYPE_* of q, k, v, out and their gradients */
  int32_t heads, q_heads, k_heads, v_heads;
  int32_t key_dim, value_dim;
  float scale; /* finite, not zero */
  int64_t batch, tokens;
  int64_t q_stride[3], k_stride[3], v_stride[3]; /* batch, token, head */
} tfa_attn_desc;

/* Device workspace (bytes) of tfa_linear_attention (backward = 0), of its backward without grad_log_decay (1) or with (2). */
int tfa_linear_attention_workspace_size(const tfa_attn_desc* desc, int32_t backward, size_t* bytes);
/* state_in may be NULL (zeros), state_out NULL (not wanted; must not be state_in otherwise). */
int tfa_linear_attention(const tfa_attn_desc* desc, const void* q, const void* k, const void* v, const float* log_decay,
                         const int64_t* lengths, const float* state_in, void* out, float* state_out, void* workspace,
                         tfa_stream stream);
/* Gradients of a loss whose gradients by out and state_out are grad_out (contiguous, as out) and grad_state_out (NULL:
 * zero).  grad_q, grad_k, grad_v: contiguous (batch, tokens, own heads, features); each gradient may be NULL, but
 * grad_log_decay needs grad_q and grad_k, and grad_state_in needs grad_v. */
int tfa_linear_attention_backward(const tfa_attn_desc* desc, const void* q, const void* k, const void* v,
                                  const float* log_decay, const int64_t* lengths, const float* state_in,
                                  const void* grad_out, const float* grad_state_out, void* grad_q, void* grad_k,
                                  void* grad_v, float* grad_log_decay, float* grad_state_in, void* workspace,
                                  tfa_stream stream);
/* One token of every stream (tokens = 1): state is updated in place, out = scale S^T q of the new state. */
int tfa_linear_attention_step(const tfa_attn_desc* desc, const void* q, const void* k, const void* v,
                              const float* log_decay, float* state, void* out, tfa_stream stream);

/*
 * Group norm with an activation on contiguous channels-last data (batch, positions, channels), 16-byte aligned:
 *   y = act((x - mean) rstd weight + bias), mean and rstd over the positions and the channels of a group
 * weight, bias: fp32 (channels) or NULL; mean, rstd: fp32 (batch, groups), written by the forward, read by the backward.
 * lengths: (batch) device int64 or NULL; positions at and past lengths[n] * inner are padding: never read, no part of the
 * statistics, zeros in y and grad_x.
 */
#define TFA_ACT_NONE 0
#define TFA_ACT_SILU 1
#define TFA_ACT_GELU 2 /* z Phi(z), by the error function */
#define TFA_ACT_RELU 3
typedef struct tfa_norm_desc {
  int32_t dtype; /* of x, y and their gradients */
  int32_t channels, groups, activation;
  int64_t batch, positions, inner;
  float eps;
  int32_t reserved;
} tfa_norm_desc;

int tfa_group_norm_workspace_size(const tfa_norm_desc* desc, int32_t backward, size_t* bytes);
int tfa_group_norm(const tfa_norm_desc* desc, const void* x, const float* weight, const float* bias,
                   const int64_t* lengths, void* y, float* mean, float* rstd, void* workspace, tfa_stream stream);
/* grad_weight and grad_bias may be NULL. */
int tfa_group_norm_backward(const tfa_norm_desc* desc, const void* x, const void* grad_y, const float* weight,
                            const float* bias, const int64_t* lengths, const float* mean, const float* rstd,
                            void* grad_x, float* grad_weight, float* grad_bias, void* workspace, tfa_stream stream);

/*
 * One AdamW step (decoupled weight decay) over many contiguous tensors:
 *   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
 *   p = p (1 - lr weight_decay) - lr / (1 - b1^step) m / (sqrt(v) / sqrt(1 - b2^step) + eps)
 * in fp32.  states: fp32, or 8-bit codes with one fp32 scale s per 256 values of a tensor: m = s sgn(c) (c / 127)^2 of int8
 * codes, v = s (c / 255)^4 of uint8 codes, s the largest magnitude of the block, c to nearest and at least 1 where v > 0.
 * With a master copy (fp32) the step is taken on it and param receives it rounded.  The tables are host memory, read before
 * the call returns.
 */
typedef struct tfa_adam_tensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale; /* 8-bit states: ceil(n / 256) scales each; else NULL */
  float* exp_avg_sq_scale;
  float* master; /* or NULL */
  int64_t n;
} tfa_adam_tensor;
typedef struct tfa_adam_desc {
  int32_t param_dtype, grad_dtype, state_bits, reserved;
  int64_t step; /* from 1 */
  double lr, beta1, beta2, eps, weight_decay;
} tfa_adam_desc;
typedef struct tfa_code_tensor {
  const void* codes;
  const float* scales;
  float* out;
  int64_t n;
} tfa_code_tensor;

int tfa_adamw_step(int64_t count, const tfa_adam_tensor* tensors, const tfa_adam_desc* desc, tfa_stream stream);
/* The fp32 values that 8-bit states stand for (squares = 0: exp_avg, 1: exp_avg_sq). */
int tfa_adamw_state_values(int64_t count, const tfa_code_tensor* tensors, int32_t squares, tfa_stream stream);

/*
 * Causal convolution along frames with a short filter for each channel, channels last, and an activation:
 *   y_t = act(bias + sum_j weight[c][j] x_{t - width + 1 + j}),  j < width
 * x: (batch, tokens, channels) at strides of batch and token (in elements; channels contiguous, any address); y and the
 * gradients are contiguous.  weight: fp32 (channels, width), bias: fp32 (channels) or NULL.  States hold the last width - 1
 * inputs, (batch, width - 1, channels) of the call's type: state_in (NULL: zeros) is what came before the first token,
 * state_out (NULL: not wanted; must not be state_in) what a sequence ends with.  lengths: (batch) device int64 or NULL; tokens at and
 * past a sequence's length are padding: never read, zeros in y and the gradients.  Sums are fp32.  Widths 1 to 8.
 */
typedef struct tfa_conv_desc {
  int32_t dtype; /* TFA_DTYPE_* of x, y, states and their gradients */
  int32_t channels, width, activation;
  int64_t batch, tokens;
  int64_t x_stride[2]; /* batch, token */
} tfa_conv_desc;

int tfa_causal_conv(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias, const int64_t* lengths,
                    const void* state_in, void* y, void* state_out, tfa_stream stream);
/* Gradients of a loss whose gradients by y and state_out are grad_y (contiguous) and grad_state_out (NULL: zero); each may be
 * NULL.  workspace: device memory of the size that tfa_causal_conv_workspace_size gives. */
int tfa_causal_conv_workspace_size(const tfa_conv_desc* desc, size_t* bytes);
int tfa_causal_conv_backward(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias,
                             const int64_t* lengths, const void* state_in, const void* grad_y, const void* grad_state_out,
                             void* grad_x, float* grad_weight, float* grad_bias, void* grad_state_in, void* workspace,
                             tfa_stream stream);
/* One token of every stream (tokens = 1): state is shifted in place. */
int tfa_causal_conv_step(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias, void* state, void* y,
                         tfa_stream stream);

/*
 * The selective scan of a state space layer, `states` values a channel:
 *   s_t = softplus(dt_t + dt_bias) (or dt_t + dt_bias),  h_t = exp(s_t a) h_{t-1} + s_t x_t b_t,
 *   y_t = (c_t . h_t + d x_t) silu(z_t)
 * x, dt, z: (batch, tokens, channels) at strides of batch and token, channels contiguous; b, c: (batch, tokens, groups, states) at
 * strides of batch, token and group, states contiguous, shared by channels / groups neighbouring channels; all of one type, at any
 * address, token strides from 0 to 2^24 - 1.  a: fp32 (channels, states), -inf for no memory; d, dt_bias: fp32 (channels) or NULL
 * (zero); z may be NULL (no gate).  State tensors are fp32 (batch, channels, states).  lengths: (batch) device int64 or NULL; tokens
 * at and past a sequence's length are padding: never read, zeros in y and the gradients, and the state is the one at the length.
 * States, exponentials and sums are fp32 for every type: a decay is rounded once a token, so over a memory of m tokens (exponents of
 * steps that are the same from token to token) a state can be off by m 2^-25 of itself.  What is not finite makes NaN or infinities
 * of its channel from its token on, but for dt_t + dt_bias of -inf under softplus: a step of 0, which leaves the state.  Up to 64
 * states.
 */
typedef struct tfa_scan_desc {
  int32_t dtype; /* TFA_DTYPE_* of x, dt, z, b, c, y and their gradients */
  int32_t channels, groups, states;
  int32_t softplus;
  int32_t bc_fixed; /* not 0: no gradients of b and c are asked of the backward, whose sums are most of its workspace */
  int64_t batch, tokens;
  int64_t x_stride[2], dt_stride[2], z_stride[2]; /* batch, token */
  int64_t b_stride[3], c_stride[3];               /* batch, token, group */
} tfa_scan_desc;

/* Bytes of the states that a backward needs of its forward, and of the workspaces of both; all 16-byte aligned device memory.  For every
 * token and channel: kept states n / 4, n being the states filled up to 4, 8, 16, 32 or 64; sums of the gradients of b and c n / 8
 * (32 at 64: two fp32 states for 16 channels). */
int tfa_selective_scan_sizes(const tfa_scan_desc* desc, size_t* kept, size_t* workspace, size_t* backward_workspace);
/* state_in may be NULL (zeros), state_out NULL (not wanted; must not be state_in), kept NULL (no backward follows). */
int tfa_selective_scan(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b, const void* c,
                       const float* d, const void* z, const float* dt_bias, const int64_t* lengths, const float* state_in,
                       void* y, float* state_out, void* kept, void* workspace, tfa_stream stream);
/* Where the gradients of a loss by y (contiguous) and state_out (NULL: zero) go; all contiguous in the layout of what they are
 * gradients of, NULL where not wanted (grad_state_in must not be grad_state_out). */
typedef struct tfa_scan_grads {
  const void* grad_y;
  const float* grad_state_out;
  void *x, *dt, *b, *c, *z;
  float *a, *d, *dt_bias, *state_in;
} tfa_scan_grads;
int tfa_selective_scan_backward(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b,
                                const void* c, const float* d, const void* z, const float* dt_bias, const int64_t* lengths,
                                const float* state_in, const void* kept, const tfa_scan_grads* grads, void* workspace,
                                tfa_stream stream);
/* One token of every stream (tokens = 1): state is updated in place. */
int tfa_selective_scan_step(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b,
                            const void* c, const float* d, const void* z, const float* dt_bias, float* state, void* y,
                            tfa_stream stream);

/*
 * The norm of all values of many contiguous tensors, norm[0] = sqrt(sum of squares) with squares summed in 64 bits, and their
 * clipping: every value times min(1, max_norm / (norm + 1e-6)), in place.  A norm that is not finite makes gradients NaN or zero.
 * tensors[d], count[d]: those of type d (TFA_DTYPE_*); host memory, read before the call returns.  norm: device fp32.
 * workspace: 8-byte aligned device memory of the size that tfa_grad_norm_workspace_size gives.  Sums are added in one order
 * whatever the timing.
 */
typedef struct tfa_grad_tensor {
  void* data;
  int64_t n;
} tfa_grad_tensor;
typedef struct tfa_grad_lists {
  const tfa_grad_tensor* tensors[3];
  int64_t count[3];
} tfa_grad_lists;
int tfa_grad_norm_workspace_size(const tfa_grad_lists* grads, size_t* bytes);
int tfa_grad_norm(const tfa_grad_lists* grads, float* norm, void* workspace, tfa_stream stream);
/* max_norm: at least 0.  Tensors must not overlap. */
int tfa_clip_grads(const tfa_grad_lists* grads, double max_norm, float* norm, void* workspace, tfa_stream stream);

/* Thread-local message describing the last failure on this thread ("" if none). */
const char* tfa_last_error(void);

/* ABI version, (major << 16) | minor. */
int32_t tfa_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* TRNFFT_AMD_H */
