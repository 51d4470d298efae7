/* bmb.h -- the C ABI of libbmb.so: a B200 (sm_100a) implementation of the
 * GEMM / attention / nn / data-parallel hot path of bare-metal-bard.
 *
 * Every entry point takes plain pointers and sizes, returns an int status
 * (0 = ok, otherwise one of BMB_E_*; bmb_last_error() gives the text for the
 * calling thread) and never takes ownership of a caller's buffer.  Pointers
 * are device pointers on the current CUDA device unless a parameter is named
 * host_*.  Calls are asynchronous on the calling thread's "current stream"
 * (bmb_set_stream; the legacy default stream unless set) except where a
 * parameter named `stream` is given or the comment says the call blocks.
 *
 * The C++ headers beside this file (kernels.h, gemm.h, flash.h, attention.h,
 * nn.h, ddp.h, gpt.h) are inline shims with the reference's own names and
 * signatures over these functions, so gpt.cu / train_gpt.cu-shaped host code
 * compiles against them unchanged.  Each declaration cites the reference
 * interface it replaces as path:line inside the reference project.
 */
#ifndef BMB_H
#define BMB_H
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BMB_OK 0
#define BMB_E_ARG 1      /* bad argument (shape, alignment, null pointer)     */
#define BMB_E_CUDA 2     /* a CUDA runtime / driver call failed               */
#define BMB_E_UNSUPPORTED 3 /* valid request this build cannot serve          */
#define BMB_E_TIMEOUT 4  /* a bounded device-side wait expired                */
#define BMB_E_NCCL 5     /* NCCL missing or an NCCL call failed               */
#define BMB_E_LIMIT 6    /* size beyond a stated maximum                      */

const char *bmb_last_error(void);
const char *bmb_version(void);
/* No counterparts in the reference.  Both replay on the host a tile schedule of the tensor-core GEMM (tile height and
 * width, whole tiles, tiles shared along K) and return 0 when every (tile, K slice) is computed exactly once.  They
 * launch nothing and are usable without a GPU.
 * bmb_gemm_plan_check: the schedule that a call with these flags takes on `ctas` SMs that hold `pairs` CTA pairs (74 on a
 * B200; half of either with BMB_GEMM_HALF_SMS), *pair_out: whether it goes to pairs, which *grid_out then counts.  (A TF32
 * product whose operands are rounded as they arrive may take 128-row tiles in its place.)
 * bmb_gemm_schedule_check: the schedule on single CTAs, whatever a call of this shape takes; with BMB_GEMM_PAIR the one of
 * 256 x 256 tiles on pairs, and `ctas` counts pairs. */
int bmb_gemm_schedule_check(int math, int flags, int batch, int M, int N, int K, int ctas,
                            int *tile_m_out, int *tile_n_out, int *whole_tiles_out, int *grid_out);
int bmb_gemm_plan_check(int math, int flags, int transA, int transB, int batch, int M, int N, int K, int ctas, int pairs, int *pair_out,
                        int *tile_m_out, int *tile_n_out, int *whole_tiles_out, int *grid_out);
/* Kernels this library has launched in this process so far (launches replayed from a CUDA
 * graph included).  No counterpart in the reference; bench.py reports it. */
long long bmb_launch_count(void);

/* ---- device-side waits that ran out ------------------------------------ */
/* No counterparts in the reference.  Every wait inside the tensor-core kernels (on a copy, on the
 * tensor core, on another role of the CTA) is bounded; when one runs out the kernel drains what it
 * has in flight, returns, and leaves a nonzero word per device that makes every later call on that device
 * which goes to such kernels return BMB_E_TIMEOUT: TF32 and BF16 products, large fp32 products, fused attention
 * (fp32 of longer sequences included) and sampling in fp32.  bmb_kernel_status reads the word of the current device
 * (0 = nothing happened).  bmb_kernel_status_clear waits for the device to go idle and resets it,
 * so that a process can carry on after it has dealt with the failed step.
 * bmb_selftest_wait_expiry exercises that path without any fault: one CTA waits at most
 * limit_cycles (1..1e8 SM clocks) on a barrier that nothing arrives on, gives up, raises the word
 * and returns; the call blocks until then and reports the cycles the wait took.  Afterwards the
 * status is set, exactly as after a real expiry, until bmb_kernel_status_clear. */
int bmb_kernel_status(int *status_out);
int bmb_kernel_status_clear(void);
int bmb_selftest_wait_expiry(long long limit_cycles, long long *host_waited_cycles);

/* ---- per-thread launch context ---------------------------------------- */
/* Stream used by every entry point without a `stream` parameter.  Thread
 * local: rank threads of one process do not disturb one another. */
int bmb_set_stream(void *cuda_stream);
void *bmb_get_stream(void);

/* Arithmetic used by bmb_gemm / bmb_batched_gemm / flash attention when the
 * caller does not say.  fp32 = SIMT FFMA, bit-comparable with the reference's
 * fp32 kernels up to summation order, or, for large single products and for
 * attention (elements from 2^-108 on), split products on the tensor cores with a smaller error than that; tf32 = tcgen05 kind::tf32 with operands
 * rounded to nearest TF32 first and fp32 accumulation in tensor memory;
 * bf16 = tcgen05 kind::f16 on bf16-rounded operands. */
#define BMB_MATH_FP32 0
#define BMB_MATH_TF32 1
#define BMB_MATH_BF16 2
int bmb_set_math_mode(int mode);   /* process wide */
int bmb_get_math_mode(void);

/* ---- registry (src/kernels.h:10-31, src/registry.cu:4-23) -------------- */
typedef void (*bmb_sgemm_fn)(int M, int N, int K, float alpha, const float *A,
                             const float *B, float beta, float *C);
typedef struct bmb_kernel_entry {
    int id;
    const char *name;
    bmb_sgemm_fn fn;
    const char *note;
    double tol; /* normwise tolerance against an fp32 reference product */
} bmb_kernel_entry;
int bmb_num_kernels(void);
const bmb_kernel_entry *bmb_kernel_table(void);
const bmb_kernel_entry *bmb_find_kernel(int id);
/* Row-major C = alpha*A@B + beta*C, the three registry kernels
 * (replaces sgemm_naive..sgemm_tensorcore, src/kernels.h:34-42). */
int bmb_sgemm_simt(int M, int N, int K, float alpha, const float *A,
                   const float *B, float beta, float *C);
int bmb_sgemm_tf32(int M, int N, int K, float alpha, const float *A,
                   const float *B, float beta, float *C);
int bmb_sgemm_bf16(int M, int N, int K, float alpha, const float *A,
                   const float *B, float beta, float *C);

/* ---- GEMM (src/gemm.h:17-19, 26-29) ----------------------------------- */
/* C[M,N] = alpha*op(A)@op(B) + beta*C, row-major, dense leading dimensions
 * exactly as src/gemm.h:6-11 defines them. */
int bmb_gemm(int transA, int transB, int M, int N, int K, float alpha,
             const float *A, const float *B, float beta, float *C,
             void *stream);
/* Same, with the arithmetic stated per call (BMB_MATH_*) and flags. */
#define BMB_GEMM_A_ROUNDED 1 /* A already holds TF32-representable values */
#define BMB_GEMM_B_ROUNDED 2 /* B already holds TF32-representable values */
#define BMB_GEMM_C_ROUNDED 4 /* store C rounded to TF32 (it feeds another tensor-core kernel) */
#define BMB_GEMM_NO_SPLIT 8  /* never split K across CTAs (keeps the summation order fixed) */
#define BMB_GEMM_TILE_M128 16 /* TF32 tensor-core path: 128-row tiles whatever the cost model says */
#define BMB_GEMM_TILE_M256 32 /* TF32 tensor-core path: 256-row tiles where the shape allows (M >= 256, N >= 256) */
#define BMB_GEMM_PAIR 64      /* tensor-core path: run on CTA pairs (tcgen05 cta_group::2, 256 x 256 tiles) where the shape allows
                                 (M >= 256, N >= 256, an M- or N-contiguous TF32 operand a multiple of 32 wide); without
                                 this flag and the next the cost model decides */
#define BMB_GEMM_NO_PAIR 128  /* tensor-core path: never use CTA pairs for this call */
#define BMB_GEMM_HALF_SMS 256 /* tensor-core path: occupy only half of the SMs (one CTA each), so that two products
                                 launched on two streams share the GPU side by side instead of one after the other */
int bmb_gemm_ex(int math, int flags, int transA, int transB, int M, int N,
                int K, float alpha, const float *A, const float *B, float beta,
                float *C, void *stream);
/* The MLP's first half in one call (no counterpart in the reference; equals gemm + bias_forward + gelu_forward of
 * src/gpt.cu:268-272): C = A W^T + bias (A [M,K], W [N,K], bias [N] or NULL, all row-major) and
 * C_gelu = GELU(C), bit-identical to bmb_gelu_forward on C.  On the tensor-core paths both leave the
 * accumulator in the product's epilogue when C and C_gelu are 16-byte aligned and N % 4 == 0 (no tile is then
 * split along K); otherwise, and for BMB_MATH_FP32, the activation is a pass of its own.
 * BMB_GEMM_AUX_ROUNDED: C_gelu is stored rounded to TF32 (it feeds another tensor-core product).
 * BMB_GEMM_AUX_FAST: where the activation rides in the epilogue, its tanh is the hardware's approximate one (absolute
 * error about 2^-11, of the order of the TF32 rounding of C_gelu; no longer bit-identical to bmb_gelu_forward). */
#define BMB_GEMM_AUX_ROUNDED 512
#define BMB_GEMM_AUX_FAST 1024
int bmb_gemm_bias_gelu(int math, int flags, int M, int N, int K, const float *A, const float *W, const float *bias,
                       float *C, float *C_gelu, void *stream);
int bmb_batched_gemm(int transA, int transB, int batch, int M, int N, int K,
                     float alpha, const float *A, long long strideA,
                     const float *B, long long strideB, float beta, float *C,
                     long long strideC, void *stream);
/* Round n floats to the nearest TF32 value (ties away from zero, the
 * cvt.rna.tf32.f32 rule the reference applies at k09_tensorcore.cu:119-128). */
int bmb_round_tf32(float *dst, const float *src, size_t n, void *stream);

/* ---- fused causal attention (src/flash.h:36-62) ------------------------ */
int bmb_flash_attention_forward(float *out, float *lse, const float *qkv,
                                int B, int T, int C, int NH);
int bmb_flash_attention_backward(float *dqkv, float *dsum, const float *dout,
                                 const float *qkv, const float *out,
                                 const float *lse, int B, int T, int C, int NH);
int bmb_flash_num_configs(void);
const char *bmb_flash_config_name(int cfg);
int bmb_flash_default_config(void);
/* status BMB_E_UNSUPPORTED <=> the reference's `false` (config cannot run for
 * this head size). */
int bmb_flash_attention_forward_cfg(int cfg, float *out, float *lse,
                                    const float *qkv, int B, int T, int C,
                                    int NH);
int bmb_flash_num_bwd_configs(void);
const char *bmb_flash_bwd_config_name(int cfg);
int bmb_flash_default_bwd_config(void);
int bmb_flash_attention_backward_cfg(int cfg, float *dqkv, float *dsum,
                                     const float *dout, const float *qkv,
                                     const float *out, const float *lse, int B,
                                     int T, int C, int NH);
/* No counterpart in the reference: the _cfg calls with a flag word.  BMB_FLASH_OPERANDS_ROUNDED
 * tells the TF32 tensor-core configuration that qkv (and dout) already hold TF32-representable
 * values, as the training step's producers leave them: the kernels then read them where they
 * lie instead of rounding copies first.  Ignored by the fp32 configurations. */
#define BMB_FLASH_OPERANDS_ROUNDED 1
int bmb_flash_attention_forward_ex(int cfg, int flags, float *out, float *lse,
                                   const float *qkv, int B, int T, int C, int NH);
int bmb_flash_attention_backward_ex(int cfg, int flags, float *dqkv, float *dsum,
                                    const float *dout, const float *qkv, const float *out,
                                    const float *lse, int B, int T, int C, int NH);

/* ---- unfused attention (src/attention.h:18-24) ------------------------- */
int bmb_attention_forward(float *out, float *qkvr, float *att,
                          const float *qkv, int B, int T, int C, int NH);
int bmb_attention_backward(float *dqkv, float *dqkvr, float *datt,
                           float *dpreatt, const float *dout,
                           const float *qkvr, const float *att, int B, int T,
                           int C, int NH);

/* ---- nn kernels (src/nn.h:10-60) -------------------------------------- */
int bmb_encoder_forward(float *out, const int *tokens, const float *wte,
                        const float *wpe, int B, int T, int C);
int bmb_encoder_backward(float *dwte, float *dwpe, const float *dout,
                         const int *tokens, int B, int T, int C);
int bmb_layernorm_forward(float *out, float *mean, float *rstd,
                          const float *inp, const float *weight,
                          const float *bias, int N, int C);
/* dinp, dweight and dbias are accumulated into (+=), as src/nn.cu:108-111. */
int bmb_layernorm_backward(float *dinp, float *dweight, float *dbias,
                           const float *dout, const float *inp,
                           const float *weight, const float *mean,
                           const float *rstd, int N, int C);
/* Same result as bmb_layernorm_backward, for callers that must not allocate.  No
 * counterpart in the reference.  A training loop that has handed all of its device memory
 * out at start-up (as gpt_alloc does) cannot afford the library's lazy cudaMalloc in the
 * middle of a step: it may fail on a full device, and it synchronises the whole device.
 * This entry point calls no cudaMalloc / cudaFree or any allocating routine: its partial
 * sums live in a fixed 4 MiB array inside the library image, present on every GPU that
 * loads libbmb.so.  Limits: C <= 1024, C % 4 == 0, 16-byte aligned buffers; a wider row
 * returns BMB_E_LIMIT.  The first call on each device looks up the array's device address
 * (once, with that device current), so make that first call before any stream capture.
 * All calls on a device share the one array: calls that overlap on the GPU (two streams,
 * two threads) race on it and must be serialised by the caller.  Nothing in the array needs
 * clearing between calls. */
int bmb_layernorm_backward_noalloc(float *dinp, float *dweight, float *dbias,
                                   const float *dout, const float *inp,
                                   const float *weight, const float *mean,
                                   const float *rstd, int N, int C);
/* No counterparts in the reference (fusions the training step uses):
 * residual_layernorm_forward: sum_out = a + b, then layernorm_forward(out, mean, rstd, sum_out, ...)
 *   (residual_forward + layernorm_forward, src/nn.cu:54-81, 152-159) in one pass over the rows.
 * layernorm_backward_colsum: layernorm_backward, and dcolsum += column sums of the updated dinp --
 *   the bias gradient (bias_backward, src/nn.cu:184-191) of the projection whose output gradient
 *   dinp is.  dcolsum may be NULL. */
/* gelu_backward over an (N x C) matrix, and dcolsum += column sums of dinp (the bias gradient
 * of the projection that produced the GELU input).  No counterpart in the reference. */
int bmb_gelu_backward_colsum(float *dinp, float *dcolsum, const float *inp,
                             const float *dout, int N, int C);
int bmb_residual_layernorm_forward(float *sum_out, float *out, float *mean, float *rstd,
                                   const float *a, const float *b, const float *weight,
                                   const float *bias, int N, int C);
int bmb_layernorm_backward_colsum(float *dinp, float *dweight, float *dbias, float *dcolsum,
                                  const float *dout, const float *inp, const float *weight,
                                  const float *mean, const float *rstd, int N, int C);
int bmb_gelu_forward(float *out, const float *inp, int n);
int bmb_gelu_backward(float *dinp, const float *inp, const float *dout, int n);
int bmb_residual_forward(float *out, const float *a, const float *b, int n);
int bmb_add_inplace(float *dst, const float *src, int n);
int bmb_bias_forward(float *out, const float *bias, int N, int C);
/* dbias += column sums of dout (src/nn.cu:184-191). */
int bmb_bias_backward(float *dbias, const float *dout, int N, int C);
int bmb_softmax_crossentropy_forward(float *probs, float *losses,
                                     const float *logits, const int *targets,
                                     int N, int V, int Vp);
int bmb_crossentropy_softmax_backward(float *dlogits, const float *probs,
                                      const int *targets, int N, int V, int Vp,
                                      float dloss_scale);
/* No counterpart in the reference: softmax_crossentropy_forward and
 * crossentropy_softmax_backward (src/nn.cu:197-237) in one sweep.  losses as
 * the forward writes them; dlogits = (softmax(logits) - onehot) * dloss_scale
 * on the V real columns, 0 on the padding.  The probabilities are not kept. */
int bmb_softmax_crossentropy_fused(float *dlogits, float *losses,
                                   const float *logits, const int *targets,
                                   int N, int V, int Vp, float dloss_scale);
int bmb_adamw_update(float *params, float *grads, float *m, float *v, int n,
                     float lr, float beta1, float beta2, float eps,
                     float weight_decay, int step, float grad_scale);
/* Blocks; *host_norm = sqrt(sum g^2) (src/nn.cu:336-355). */
int bmb_grad_global_norm(const float *grads, int n, float *host_norm);
int bmb_zero_buffer(float *p, size_t n);
/* Blocks; *host_mean = mean of n device values (src/nn.cu:359-368). */
int bmb_reduce_mean(const float *d_values, int n, float *host_mean);

/* Device-resident variants used by the training step so that a step has no
 * host round trip: the squared norm and the loss stay on the device, and the
 * optimiser derives its clip factor from the device value.
 * sumsq_out[0] = sum g^2 (double).  */
int bmb_grad_sumsq_device(const float *grads, size_t n, double *sumsq_out);
int bmb_reduce_mean_device(const float *d_values, int n, float *d_mean);
/* grad_scale = (norm/div > clip ? clip/(norm/div) : 1)/div with
 * norm = sqrt(*d_sumsq), the rule of src/train_gpt.cu:442-448 (div = ranks).
 * shadow (may be null) receives the TF32-rounded copy of the new params. */
int bmb_adamw_update_clipped(float *params, const float *grads, float *m,
                             float *v, size_t n, float lr, float beta1,
                             float beta2, float eps, float weight_decay,
                             int step, const double *d_sumsq, float clip,
                             float div, float *shadow);

/* ---- serving several requests: a paged cache, attention over it, logits before a draw ------------ */
/* No counterparts in the reference, whose generate() (src/train_gpt.cu:46-102) serves one text.  A step of a program that
 * answers several requests at once is: bmb_pages_assign (pages and slots for the step's new tokens), per layer
 * bmb_paged_kv_write and bmb_paged_attention, bmb_logits_adjust before the draw, and bmb_pages_release for requests that end.
 * None of them allocates, blocks or keeps anything between calls, so all can be captured; sums and softmax statistics are fp32.
 *
 * A cache is a pool of pages of page_size tokens each.  Token t of page p has its keys of head h at
 * k + p * page_stride + t * token_stride + h * head_stride (strides in elements; head_size elements in a row), its values at
 * the same place of v: [pages][page_size][heads][head_size] and [pages][heads][page_size][head_size] alike, k and v apart or
 * interleaved.  Both pointers and all strides are multiples of 16 bytes, every stride at least head_size; head_size is
 * 32, 64 or 128 (BMB_E_UNSUPPORTED otherwise); pages * page_size fits an int (BMB_E_LIMIT).  The slot of that token is
 * p * page_size + t.  The struct is read during the call only. */
#define BMB_TYPE_FP32 0
#define BMB_TYPE_BF16 1
#define BMB_TYPE_FP16 2
typedef struct bmb_kv_cache {
    void *k, *v;
    long long page_stride, token_stride, head_stride;
    int type; /* BMB_TYPE_* of the elements */
    int pages, page_size, heads, head_size;
} bmb_kv_cache;

/* Pages for the new tokens of n requests, and the slot of each.  Request i has lens[i] tokens in the cache, in the pages of
 * row i of tables ([n][max_pages]), and gets new_lens[i] more (negative: 0; 1 in a step of decoding, many for a prompt, 0 for
 * a request that rests).  Pages are popped from the stack free_pages[0 .. *free_count) (clamped to `pages`, the size of the
 * pool and of that array), from its end, in the order of the requests.  A request that the pool cannot serve, that
 * would need more than max_pages or whose tokens end beyond max_tokens gets nothing (lens_out tells); after the first
 * request that the pool cannot serve only those that need no page are served.
 *   tables     the entries of new pages are written, others are left alone
 *   lens_out   [n] lens + new_lens, or lens where the request was not served (may be lens itself)
 *   slots      [max_tokens] of the new tokens, request after request; -1 for tokens of requests not served, for tokens whose
 *              page is not one of the pool, and behind the last token (where positions is 0 and owners -1)
 *   positions  [max_tokens] a token's index in its request, owners [max_tokens] the request (each may be NULL)
 *   starts     [n + 1] where each request's tokens begin and the last one's end, at most max_tokens (may be NULL)
 *   free_left  pages left on the stack (may be free_count itself); free_pages is not written
 * All pointers are device pointers, lens and new_lens included; sums of lengths are 64-bit.  Here and in bmb_pages_release n is at most 2^31 - 1024
 * and a pool's tokens and those of a row of the tables fit an int (BMB_E_LIMIT). */
int bmb_pages_assign(int *tables, int *lens_out, int *slots, int *positions, int *owners, int *starts, int *free_left,
                     const int *lens, const int *new_lens, const int *free_pages, const int *free_count, int n, int max_pages,
                     int page_size, int pages, int max_tokens, void *stream);
/* The pages of the requests with done[i] != 0 go back on the stack, request after request and in the order of their tables:
 * written from free_pages[*free_count] on, *free_out = the new count (may be free_count itself), lens_out[i] = 0 for
 * those and lens[i] (at least 0) for the others (may be lens itself).  Entries that are not pages of the pool are left out, and what the stack
 * (`pages` entries) has no room for.  tables is not written; a page must not be in two tables. */
int bmb_pages_release(int *free_pages, int *free_out, int *lens_out, const int *free_count, const int *lens, const int *tables,
                      const int *done, int n, int max_pages, int page_size, int pages, void *stream);
/* Rows of keys and values (heads * head_size floats each, row_stride floats from one token to the next: 3C for rows of a qkv
 * product) into the slots of their tokens, rounded to the cache's type (to nearest even; beyond fp16's range: infinity).
 * Rows whose slot is negative or beyond the pool are left out (but are there: all `tokens` rows may be read).  Slots are distinct (of two rows with one slot either may be
 * found there, or elements of both). */
int bmb_paged_kv_write(const bmb_kv_cache *cache, const float *k, const float *v, long long row_stride, const int *slots,
                       int tokens, void *stream);
/* Attention of one new token of each of n requests over the tokens that the cache holds of it (its own included, once written):
 * out[i][h] = sum_j softmax_j(scale q[i][h] . k_j) v_j over j < lens[i] (clamped to the table), where heads is a multiple of the
 * cache's and query head h reads cache head h / (heads / cache->heads).  Rows of q and out are q_stride and out_stride floats
 * apart, row i being request i's (q may lie in rows of a qkv product, if these are one for each request, as where each adds one token in a step;
 * otherwise request i's newest token is in row starts[i + 1] - 1 of the new tokens', and q is gathered from there; out must not overlap q).  lse ([n][heads], may be NULL) receives the natural
 * logarithm of the sum of exponentials.  Row i of tables ([n][max_pages]) names request i's pages; tokens in pages that are
 * not of the pool count as absent, and are not read.  Where nothing is left, out is 0 and lse -infinity.
 * workspace: bmb_paged_attention_workspace bytes on the device, 16-byte aligned, of this call's own until it has run (two
 * streams, or two graphs that may run at once, have one each); its contents need no preparation and mean nothing afterwards.
 * Products and sums are of fp32 accuracy whatever the cache's type (with an fp16 cache elements of q are kept to 2^-39 of their row's
 * largest, with an fp32 cache elements of q, keys and values to 2^-136, where their second pieces end).
 * Infinities and NaN in q, and in keys and values that count, do what they do in fp32 in sum_j w_j v_j / sum_j w_j, w_j = exp(s_j - max s): a
 * score of NaN or +infinity makes a head's outputs and lse NaN, a score of -infinity has weight 0 (where no other token counts, nothing is left), an
 * infinite value makes its column infinite, or NaN beside the other infinity or with a weight that is 0.  Finite inputs have finite outputs as long as q . k, s / ln 2 and
 * sum_j w_j |v_j| are in fp32's range. */
/* bmb_paged_attention_schedule_check replays on the host how a call of `blocks` thread blocks (at most 512) divides its work (launches nothing, no GPU needed) and
 * returns 0 when every tile of every head is worked on exactly once and every part is joined; *joined_out: heads whose parts lie
 * in several blocks.  max_len: max_pages * page_size. */
int bmb_paged_attention_schedule_check(const int *host_lens, int n, int heads, int kv_heads, int head_size, int type, int max_len,
                                       int blocks, long long *tiles_out, int *joined_out);
size_t bmb_paged_attention_workspace(int heads, int kv_heads, int head_size);
int bmb_paged_attention(float *out, float *lse, const float *q, const bmb_kv_cache *cache, const int *tables, const int *lens,
                        int n, int heads, long long q_stride, long long out_stride, int max_pages, float scale, void *workspace,
                        size_t workspace_bytes, void *stream);

/* Rules for rows of logits, each part optional (NULL), every array on the device:
 *   history   [n][history_stride] tokens of each text, the first history_lens[i] count, of those the first prompt_lens[i]
 *             (NULL: none) are the prompt; entries outside the vocabulary are passed over
 *   repetition, frequency, presence   [n], need history
 *   bias_ids, bias   [n][bias_stride], the first bias_lens[i] count; of entries for one token the last; ids outside the vocabulary are passed over
 *   allowed   [n][allowed_stride] words: bit v % 32 of word v / 32 is 1 where token v may be drawn
 * Lengths are clamped to their strides.  Rows are there to their strides' ends: what is behind a length may be read, and means nothing. */
typedef struct bmb_logit_rules {
    const int *history, *history_lens, *prompt_lens;
    const float *repetition, *frequency, *presence;
    const int *bias_ids;
    const float *bias;
    const int *bias_lens;
    const unsigned *allowed;
    int history_stride, bias_stride, allowed_stride;
} bmb_logit_rules;
/* out[i][v] for v < V, rows of both `stride` floats apart (out may be logits itself), in this order:
 *   x = logits;  v in the text: x > 0 ? x / repetition : x * repetition;  v drawn: x -= frequency * (times v was drawn), x -= presence;
 *   v among the biases: x += bias;  not allowed: -infinity
 * every step rounded to fp32 by itself.  Columns from V on are left as they are in out.  A row whose mask allows nothing is -infinity
 * throughout. */
int bmb_logits_adjust(float *out, const float *logits, int n, int V, long long stride, const bmb_logit_rules *rules, void *stream);

/* ---- data-parallel all-reduce (src/ddp.h:32-69) ------------------------ */
typedef struct bmb_ddp_timing {
    double reduce_scatter_ms;
    double all_gather_ms;
    double total_ms;
    size_t bytes_per_device;
} bmb_ddp_timing;

/* Single-process form, one rank per entry of `devices` (a device may repeat,
 * src/ddp.h:53-57).  The handle is opaque; the C++ shim keeps it inside the
 * reference-shaped DDP struct. */
typedef struct bmb_ddp bmb_ddp;
int bmb_ddp_create(bmb_ddp **out, int n, const int *devices);
int bmb_ddp_destroy(bmb_ddp *d);
/* In-place sum over ranks of bufs[r][0..count); blocks until complete. */
int bmb_ddp_allreduce(bmb_ddp *d, float **bufs, size_t count);
int bmb_ddp_timing_get(const bmb_ddp *d, bmb_ddp_timing *out);
/* The part of a count-element buffer that rank r reduces and then serves to
 * the others: ceil(count/n) elements from r*ceil(count/n), clipped to the end
 * (the chunking of src/ddp.cu:34-40).  Host-only arithmetic. */
int bmb_ddp_slice(size_t count, int n, int r, size_t *off_out, size_t *len_out);
/* peer[i*n+j] = 1 when rank i reaches rank j's memory directly. */
int bmb_ddp_peer_matrix(const bmb_ddp *d, int *n_out, int *dev_out,
                        unsigned char *peer_out);
int bmb_ddp_report_topology(const bmb_ddp *d);

/* One-process-per-GPU form (NCCL over NVLink/NVSwitch; libnccl.so.2 is
 * opened on first use).  id is the 128-byte NCCL unique id made by rank 0 and
 * handed to every rank by the launcher. */
typedef struct bmb_comm bmb_comm;
int bmb_comm_unique_id(unsigned char id_out[128]);
int bmb_comm_create(bmb_comm **out, const unsigned char id[128], int nranks,
                    int rank);
int bmb_comm_destroy(bmb_comm *c);
/* In-place sum of count floats over all ranks, asynchronous on `stream`. */
int bmb_comm_allreduce(bmb_comm *c, float *buf, size_t count, void *stream);
int bmb_comm_allreduce_f64(bmb_comm *c, double *buf, size_t count, void *stream);

/* ---- GPT training step (caller of all of the above; src/gpt.h:10-79,
 *      src/train_gpt.cu:397-464) ---------------------------------------- */
typedef struct bmb_trainer bmb_trainer;
typedef struct bmb_train_config {
    int max_seq_len, vocab_size, padded_vocab, n_layer, n_head, n_embd;
    int B, T;          /* per-rank batch and sequence length               */
    int use_flash;     /* 1 fused attention, 0 the unfused path             */
    int math;          /* BMB_MATH_* for the GEMMs and attention            */
    int fused;         /* 1 = fused epilogues, 0 = the reference's op list  */
    float beta1, beta2, eps, weight_decay, grad_clip;
} bmb_train_config;
int bmb_trainer_create(bmb_trainer **out, const bmb_train_config *cfg,
                       unsigned seed);
int bmb_trainer_destroy(bmb_trainer *t);
int bmb_trainer_attach_comm(bmb_trainer *t, bmb_comm *c, int nranks);
/* Fused gradient exchange + optimiser over peer memory (one process per GPU, 2..8 ranks; replaces
 * ddp_allreduce + grad norm + adamw_update of src/train_gpt.cu:431-451 inside bmb_trainer_step):
 * rank r owns the r-th of n equal pieces of every tensor (of every layer group of a stacked tensor); it
 * sums its pieces of all ranks' gradients by reading the peers' buffers, the ranks add their squared
 * norms, every rank updates its pieces and stores the new parameters into all ranks' buffers.  All of it
 * runs on a second (exchange) stream, so bmb_trainer_step returns with the exchange still in flight; the
 * next step and every other entry point wait for it first.  BMB_TRAINER_OVERLAP=1 exchanges the parameter
 * space in three chunks (embeddings + layer 0 | the first half of the other layers | the second half + final
 * layernorm) and sums a chunk's gradients as soon as backward has finished them; =2 also lets the next step's
 * forward begin on the chunks that have arrived.  Both measured no faster than the default at 2 and 4 GPUs.
 * bmb_trainer_ipc_export writes this rank's 192-byte handle record; the launcher
 * gathers the records of all ranks in rank order and hands them to bmb_trainer_attach_peers
 * (after bmb_trainer_attach_comm, whose communicator carries the small collectives that order
 * the phases).  records = NULL detaches (back to the communicator's all-reduce); all ranks must
 * attach or none.  After a fused step bmb_trainer_get_grads returns summed values only inside
 * this rank's pieces. */
int bmb_trainer_ipc_export(bmb_trainer *t, void *record192);
int bmb_trainer_attach_peers(bmb_trainer *t, int rank, int nranks, const void *records);
/* The step's plan for a configuration (host only, no GPU needed; no counterpart in the reference): the chunks
 * as ranges of the flat parameter space -- ranges[(chunk * 16 + i) * 2 + {0, 1}] = offset, length in floats,
 * nranges[chunk] of them, 3 chunks -- and the pieces the step is captured in: pieces[4 * i + {0..3}] = first
 * unit, end unit, chunk whose update the piece waits for (-1: none), chunk whose gradients are final when it ends
 * (-1: none); units are 0 embedding, 1 + l layer l, L + 1 head and loss, L + 2 head backward, 2L + 2 - l layer
 * l backward, 2L + 3 embedding backward.  overlapped = 0 gives the single-chunk, single-piece plan. */
int bmb_trainer_step_plan(const bmb_train_config *cfg, int overlapped, unsigned long long *ranges /* [3][16][2] */,
                          int *nranges /* [3] */, int *pieces /* [5][4] */, int *npieces);
size_t bmb_trainer_num_params(const bmb_trainer *t);
int bmb_trainer_get_params(bmb_trainer *t, float *host_out);
int bmb_trainer_set_params(bmb_trainer *t, const float *host_in);
int bmb_trainer_get_grads(bmb_trainer *t, float *host_out);
/* Make tokens/targets (B*T ints each) the resident batch: an asynchronous copy on the trainer's
 * stream from host memory (pinned or pageable) or from device memory where a batch was staged. */
int bmb_trainer_upload(bmb_trainer *t, const int *host_tokens,
                       const int *host_targets);
/* One optimiser step on the resident batch: forward, backward, gradient
 * all-reduce (if a comm is attached), global-norm clip, AdamW.  Asynchronous;
 * the mean loss of the step lands in a device scalar. `step` counts from 1. */
int bmb_trainer_step(bmb_trainer *t, float lr, int step);
/* Forward+backward only (gradients left in place), for gradient parity. */
int bmb_trainer_forward_backward(bmb_trainer *t);
/* Blocks: waits for the stream and returns the last step's mean loss. */
int bmb_trainer_loss(bmb_trainer *t, float *host_loss);
/* The same read without the wait: enqueues the 4-byte device-to-host copy of the last step's mean
 * loss on the trainer's stream and returns; `pinned_host_loss` must be page-locked and is valid once
 * the stream has passed this point (an event recorded after the call, or bmb_trainer_sync).  Lets a
 * training loop read every step's loss one step late instead of draining the GPU every step. */
int bmb_trainer_loss_async(bmb_trainer *t, float *pinned_host_loss);
int bmb_trainer_sync(bmb_trainer *t);
/* Floats held by one replica: parameters (x4 with gradients and the two AdamW moments), forward
 * activations, backward scratch -- the figures the reference prints before training and under
 * --alloc-only (src/train_gpt.cu:339-355).  The per-device scratch that all callers share is not counted; in fp32
 * mode it holds 6 bytes per operand element of the largest product, until the last fp32 trainer is destroyed. */
int bmb_trainer_memory(const bmb_trainer *t, size_t *param_floats, size_t *activation_floats,
                       size_t *scratch_floats);
/* Blocks: the gradient norm the last bmb_trainer_step clipped against, ||sum over ranks of g|| / ranks
 * (src/train_gpt.cu:442-446). */
int bmb_trainer_grad_norm(bmb_trainer *t, float *host_norm);
/* Blocks: forward pass only on the resident batch, mean loss returned (the evaluate() of
 * src/train_gpt.cu:163-173 calls gpt_forward this way).  Parameters and gradients are untouched. */
int bmb_trainer_forward_loss(bmb_trainer *t, float *host_loss);

/* ---- GPT1 checkpoints and sampling (src/train_gpt.cu:175-227, 46-102) ---- */
/* Write the parameters in the reference's GPT1 layout: int32 magic 0x47505431, the six int32 of GPTConfig,
 * int32 nvocab, nvocab bytes mapping token id -> character, then num_params fp32 in the reference's tensor
 * order.  A file written here loads in the reference's `train_gpt --load` and the other way round.
 * with_optimizer_state != 0 appends what the reference does not keep -- int32 magic 0x4F424D42, int32 step,
 * the AdamW first and second moments -- after the point where the reference's reader stops. */
int bmb_trainer_save(bmb_trainer *t, const char *path, const char *itos, int nvocab,
                     int with_optimizer_state, int step);
/* Read a GPT1 file's header: fills the six model fields of *cfg_out (the others are left alone), the
 * vocabulary (at most itos_cap bytes of it), whether the optimiser-state section is present and its step. */
int bmb_checkpoint_header(const char *path, bmb_train_config *cfg_out, int *nvocab_out, char *itos_out,
                          int itos_cap, int *has_optimizer_state, int *step_out);
/* Load parameters (and, if asked, the optimiser state and *step_out) into a trainer whose six model fields
 * equal the file's; BMB_E_ARG otherwise, or when the state is asked for and absent. */
int bmb_trainer_load(bmb_trainer *t, const char *path, int load_optimizer_state, int *step_out);
/* Forward pass on host_tokens (B*T ints) and the softmax of row `pos` (0 <= pos < B*T) of the logits:
 * host_probs receives padded_vocab floats, zeros on the padding (what src/train_gpt.cu:73-78 reads). Blocks. */
int bmb_trainer_next_token_probs(bmb_trainer *t, const int *host_tokens, int pos, float *host_probs);
/* The reference's generate(): starts from start_token, draws `steps` tokens with mt19937(seed) and a
 * uniform float per token, probabilities raised to 1/temperature and renormalised when temperature != 1,
 * the window sliding once the context is full.  host_tokens_out receives the drawn token ids. Blocks.
 * Where the largest probability's power 1 / temperature is below fp32's normal numbers (where the reference divides by a sum of 0 and draws the last token), powers
 * are those of shares of the largest, so that a cold draw is of the likeliest tokens. */
int bmb_trainer_generate(bmb_trainer *t, int start_token, int steps, unsigned seed, float temperature,
                         int *host_tokens_out);
/* Several texts at once: text i begins with the host_prompt_lens[i] (at least 1) tokens of row i of host_prompts ([n][prompt_stride]) and draws
 * `steps` tokens as bmb_trainer_generate does, with mt19937(seed + i), from logits that the penalties have gone over (bmb_logits_adjust over
 * its prompt and what it drew; 1, 0, 0: none).  A text that draws stop_token ends with it (-1: none does).  host_tokens_out ([n][steps]) receives
 * the draws, -1 behind a text's end.  Prompts go through the model in one pass, then a row for each text and step, with keys and values
 * of cache_type in pages (bmb_pages_assign to bmb_pages_release above).  Each prompt and its draws fit the model's positions
 * (BMB_E_LIMIT): there is no sliding window.  Head sizes 32, 64 and 128.  Blocks; memory is taken for the call and given back.  Probabilities
 * are bmb_trainer_generate's up to rounding (of cache_type's, for keys and values). */
typedef struct bmb_batch_sampling {
    float temperature, repetition, frequency, presence;
    int stop_token, cache_type;
} bmb_batch_sampling;
int bmb_trainer_generate_batch(bmb_trainer *t, int n, const int *host_prompts, int prompt_stride, const int *host_prompt_lens, int steps,
                               unsigned seed, const bmb_batch_sampling *how, int *host_tokens_out);
/* The CUDA stream every step of this trainer is enqueued on (for events). */
void *bmb_trainer_stream(bmb_trainer *t);
/* Per-call event timing of the GEMMs inside steps (on = 1 / off = 0); the
 * totals since the last reset: flop count, device milliseconds, launches. */
int bmb_trainer_profile(bmb_trainer *t, int on);
int bmb_trainer_profile_read(bmb_trainer *t, double *gemm_flop,
                             double *gemm_ms, long long *gemm_calls,
                             long long *kernel_launches);

#ifdef __cplusplus
}
#endif
#endif /* BMB_H */
