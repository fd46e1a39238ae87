/* arke_b200 — C ABI of the B200 (sm_100a) kernels behind Arke's backend / runner interfaces.
 *
 * Conventions for every entry point
 *   - plain device pointers and sizes; the caller owns every buffer (inputs, outputs, workspaces);
 *   - nothing here allocates, frees or synchronises: work is enqueued on `stream` (a cudaStream_t
 *     passed as void*, NULL = legacy default stream) of the calling thread's current device;
 *   - returns ARKE_OK (0) or a negative ARKE_ERR_* code; arke_b200_last_error() returns the
 *     message of the calling thread's last failure;
 *   - row strides (`ld*`) are in elements;
 *   - kernels with device-side waits bound every wait; if one expires the kernel records a
 *     non-zero code in a per-device status word that arke_b200_kernel_status() reads back.
 *
 * The reference (blueyi/arke) is pure Python and has no FFI of its own; each entry point below
 * replaces the kernel that Arke's code-generating backends would have produced for the op, and
 * is reached from Python through ArkeBackend.run (arke/backend/protocol.py:94-137) /
 * BaselineRunner.get_fn (benchmarks/baselines/base.py:18-114).
 */
#ifndef ARKE_B200_H
#define ARKE_B200_H

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define ARKE_B200_API __attribute__((visibility("default")))
#else
#define ARKE_B200_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
enum { ARKE_BF16 = 0, ARKE_F16 = 1, ARKE_F32 = 2, ARKE_I8 = 3, ARKE_E4M3 = 4, ARKE_I32 = 5, ARKE_I64 = 6 };
/* quantised output kinds of quantize_per_token */
enum { ARKE_QUANT_INT8 = 0, ARKE_QUANT_E4M3 = 1 };
/* layout of the GEMM weight operand */
enum { ARKE_W_KN = 0 /* W[K,N], N contiguous */, ARKE_W_NK = 1 /* W[N,K], K contiguous */ };

/* status codes */
enum {
  ARKE_OK = 0,
  ARKE_ERR_ARG = -1,       /* null pointer / bad enum value            */
  ARKE_ERR_DTYPE = -2,     /* unsupported element type                 */
  ARKE_ERR_SHAPE = -3,     /* unsupported shape or stride              */
  ARKE_ERR_ALIGN = -4,     /* pointer or stride not aligned as needed  */
  ARKE_ERR_CUDA = -5,      /* a CUDA runtime / driver call failed      */
  ARKE_ERR_WORKSPACE = -6, /* workspace too small                      */
  ARKE_ERR_DEVICE = -7,    /* device is not sm_100                     */
  ARKE_ERR_KERNEL = -8     /* a kernel reported an expired wait        */
};

/* Library version string, e.g. "arke_b200 0.1 (sm_100a)". */
ARKE_B200_API const char* arke_b200_version(void);
/* Message of the calling thread's most recent failing call ("" if none). */
ARKE_B200_API const char* arke_b200_last_error(void);
/* Reads and clears the current device's kernel status word (synchronises `stream`).
 * 0 = nothing to report; otherwise the first code a kernel recorded: 1..5 = a bounded wait expired
 * (TMA producer, MMA issuer, epilogue, softmax, correction), 6 = arke_b200_fused_linear_ce over
 * the whole vocabulary met a label outside [0, V) (that row's loss is NaN), 7 = a library built
 * with -DARKE_B200_CHECKED computed a global index outside its extent (the access was skipped),
 * 8 = a paged entry point met a page, length or position outside its range (see there). */
ARKE_B200_API int arke_b200_kernel_status(void* stream);

/* Failure-path self-test: launches one CTA that waits on a barrier nothing completes, with a
 * limit of `limit_cycles` SM cycles (<= 2e9); the wait expires, the kernel records a non-zero code
 * in the status word exactly like the production kernels and returns normally (no trap, the
 * context stays usable).  arke_b200_kernel_status() then returns that code.  No reference
 * counterpart. */
ARKE_B200_API int arke_b200_selftest_wait_timeout(int64_t limit_cycles, void* stream);

/* Checked build (nvcc -DARKE_B200_CHECKED, `python -m arke_b200.build --flag=-DARKE_B200_CHECKED
 * --out ...`): every kernel re-derives, right before a global access, that the element index it
 * computed lies inside the tensor and otherwise records status code 7 and skips the access.  It
 * stands in for an address sanitizer where none can run.  This self-test evaluates the check on an
 * index one past an extent without touching memory: after it arke_b200_kernel_status() returns
 * 7.  ARKE_ERR_ARG in a default build.  No reference counterpart. */
ARKE_B200_API int arke_b200_selftest_bounds_check(void* stream);

/* Per-thread tuning options for the calls this thread makes afterwards (value 0 restores the
 * library's own choice).  They are what the backend maps the agent loop's strategy decisions to
 * (`lower(graph, strategy=...)`, arke/backend/llvm_backend.py:238-262, arke/ir/strategy.py:368-396):
 *   "gemm_tile_m"   128 = one-CTA 128 x 256 tiles, 256 = CTA-pair 256 x 256 tiles (cta_group::2);
 *                   applies to quant_gemm, matmul and fused_linear_ce
 *   "gemm_band_mb"  MB of the A operand kept L2-resident per band of output tiles (default 32)
 *   "gemm_static_sched" 1 = the CTA pairs of a GEMM take their tiles round robin; 0 = default:
 *                   from a device counter, so that the tiles in flight are always neighbours in
 *                   the tile order and pairs that share an operand tile through the L2 use it
 *                   at the same time
 *   "gemm_no_pdl"   1 = launch the GEMM kernels without programmatic stream serialization (their
 *                   set-up then no longer overlaps the tail of the previous kernel); 0 = default
 *   "gemm_no_split" 1 = the last, partly filled wave of a CTA-pair GEMM keeps whole 256 x 256
 *                   tiles; 0 = default: those tiles are cut into 2 or 4 narrower units along N
 *                   so that they spread over more CTA pairs
 *   "paged_prefix_kb" KB of re-read keys and values from which on a shared prefix of paged_gqa_fwd is
 *                   computed apart, once for all sequences (0 = default, 40960); set it before the
 *                   workspace is asked for
 * Results do not depend on the gemm options; paged_prefix_kb changes in which order partial sums meet.
 * get_option returns -1 for an unknown name. */
ARKE_B200_API int arke_b200_set_option(const char* name, int64_t value);
ARKE_B200_API int64_t arke_b200_get_option(const char* name);

/* Per-token (per-row) symmetric quantisation.
 * Replaces the kernels generated for `quantize_per_token`
 * (arke/ir/ops/reference_impls.py:215-218; arke/backend/triton_templates/quantize.py.j2:16-101).
 *   x [M,N] bf16/f16/f32, row stride ldx.  q [M,N] int8 or e4m3 bytes, row stride ldq.
 *   formula 0: scale = amax/127 (int8) or amax/448 (e4m3); q = rint(x/scale) with a correctly
 *              rounded fp32 quotient, half-to-even, clamp [-128,127]; all-zero rows give q = 0.
 *   formula 1: int8 only, the benchmark driver's golden (benchmarks/bench_l1.py:443-448):
 *              q = round(h(h(x/amax)*127)), h = round to the input dtype; scale out = amax. */
ARKE_B200_API int arke_b200_quantize_per_token(const void* x, int x_dtype, int64_t M, int64_t N, int64_t ldx,
                                 void* q, int64_t ldq, float* scale, int out_kind, int formula,
                                 void* stream);

/* Per-channel dequantisation  Y[i,j] = (X[i,j] - zero_point[j]) * scale[j]  in fp32
 * (`dequantize_per_channel`, arke/ir/ops/reference_impls.py:220-224; schema catalog.py:468-479).
 *   x [M,N] int8; scale [N] fp32; zero_point [N] fp32 or NULL (= 0); y [M,N] f32 / bf16 / f16.
 * (Inside the W8A8 path this scaling is fused into the GEMM epilogue; this entry point serves the
 * stand-alone catalog op.) */
ARKE_B200_API int arke_b200_dequantize_per_channel(const void* x, int64_t M, int64_t N, int64_t ldx, const float* scale,
                                     const float* zero_point, void* y, int y_dtype, int64_t ldy,
                                     void* stream);

/* RMSNorm with optional residual add and optional fused per-token quantisation of the result:
 *   h = x (+ residual);  y = T(h / sqrt(mean(h^2) + eps) * w)
 * (`rmsnorm`, arke/ir/ops/reference_impls.py:85-90; `rmsnorm_residual`, the function after
 * ref_gelu_and_mul in the same file; schemas arke/ir/ops/catalog.py:229-239,414-424).
 *   x, residual (may be NULL) [M,N], w [N]: one dtype (bf16/f16/f32).  y [M,N] same dtype or NULL.
 *   q [M,N] int8 / e4m3 bytes + scale [M] (out_kind as in quantize_per_token) or NULL: the
 *   quantisation of the rounded y, exactly what quantize_per_token would produce from it. */
ARKE_B200_API int arke_b200_rmsnorm(const void* x, const void* residual, const void* w, int dtype, int64_t M,
                      int64_t N, int64_t ldx, int64_t ldr, float eps, void* y, int64_t ldy, void* q,
                      int64_t ldq, float* scale, int out_kind, void* stream);

/* Rotary position embedding, rotate-half form (`rope`, arke/ir/ops/reference_impls.py:197-206;
 * schema arke/ir/ops/catalog.py:425-435):
 *   y[..., :D/2] = x1*cos - x2*sin,   y[..., D/2:] = x2*cos + x1*sin
 *   x, y contiguous [B,H,S,D]; cos, sin contiguous [S,D/2]; one dtype for all (bf16 / f16 / f32).
 * Every product and sum is rounded to that dtype, like the interpreter's eager evaluation, so the
 * result is bit-identical to it.  D must be even. */
ARKE_B200_API int arke_b200_rope(const void* x, const void* cos, const void* sin, void* y, int dtype,
                   int64_t B, int64_t H, int64_t S, int64_t D, void* stream);

/* The step between a packed QKV projection and attention in one pass: qkv [B*S, ld] holds, per
 * token, Hq query heads, then Hkv key heads, then Hkv value heads of D values each; Q and K heads
 * get `rope` at position s, V is copied, and all three are written in the [B,H,S,D] layout that
 * `grouped_query_attention` reads (arke/ir/ops/reference_impls.py:236-244).  This is the fused
 * form of the QKV-projection -> rope -> attention slot the reference's fusion harness reserves
 * (benchmarks/bench_l2.py:1135-1191 runs it unfused and without rope).
 *   q [B,Hq,S,D], k, v [B,Hkv,S,D] contiguous; cos, sin [S,D/2]; one dtype for all. */
ARKE_B200_API int arke_b200_qkv_rope_split(const void* qkv, int64_t ld, const void* cos, const void* sin,
                             void* q, void* k, void* v, int dtype, int64_t B, int64_t S,
                             int64_t Hq, int64_t Hkv, int64_t D, void* stream);

/* Device self-test of the quantisation kernels' fast quotient: for every finite 16-bit input
 * value x and every 16-bit row maximum amax >= |x| in [2^-60, 2^60] (rows outside that range
 * take the division path) it compares the quantised code obtained from the three-instruction
 * corrected quotient x / RN(amax / d) (d = 127 for int8, 448 for e4m3) with the code obtained
 * from the IEEE division the reference performs.  counters[0] = mismatching pairs (must be 0), counters[1] = pairs
 * checked; `counters` is device memory for two 64-bit integers.  No reference counterpart. */
ARKE_B200_API int arke_b200_selftest_quant_division(int x_dtype, int out_kind, unsigned long long* counters,
                                      void* stream);

/* Packed SwiGLU: Y = silu(X[:, :N]) * X[:, N:]  (arke/ir/ops/reference_impls.py:167-171;
 * arke/backend/triton_templates/gated_activation.py.j2:21-92), optionally fused with per-row
 * e4m3 re-quantisation of Y (scale = amax|Y| / 448).
 *   x [M,2N] bf16/f16/f32.  y [M,N] same dtype as x, or NULL.  yq [M,N] e4m3 bytes + scale [M],
 *   or NULL.  At least one of y / yq must be given. */
ARKE_B200_API int arke_b200_silu_and_mul(const void* x, int x_dtype, int64_t M, int64_t N, int64_t ldx, void* y,
                           int64_t ldy, void* yq, int64_t ldq, float* scale, void* stream);

/* Quantised GEMM with per-row x per-channel dequantisation:
 *   acc[i,j] = sum_k A[i,k] * W[k,j]   (int8 x int8 -> int32 exact, or e4m3 x e4m3 -> fp32)
 *   Y[i,j]   = out_dtype((float(acc) * sa[i]) * sw[j])
 * Composition of quantize_per_token, matmul and dequantize_per_channel
 * (arke/ir/ops/reference_impls.py:118-119, 215-224; arke/ir/ops/catalog.py:70-80,458-479).
 *   a [M,K] K-contiguous (row stride lda); w per w_layout (row stride ldw);
 *   sa [M], sw [N] fp32 (either may be NULL = 1.0);
 *   y [M,N] bf16/f16/f32 (NULL to skip), acc_out [M,N] int32 or fp32 raw accumulators (NULL to skip).
 *   ab_dtype: ARKE_I8 or ARKE_E4M3. */
ARKE_B200_API int arke_b200_quant_gemm(const void* a, int64_t lda, const void* w, int64_t ldw, int w_layout,
                         int ab_dtype, const float* sa, const float* sw, int64_t M, int64_t N,
                         int64_t K, void* y, int y_dtype, int64_t ldy, void* acc_out,
                         int64_t ldacc, void* stream);

/* Dense GEMM  C[M,N] = A[M,K] * B  with fp32 accumulation (the `matmul` op,
 * arke/ir/ops/reference_impls.py:118-119).  a, b, c: bf16, f16 or f32 (same dtype); f32 operands
 * are multiplied as TF32 (10-bit significand) on the tensor cores, which stays inside the
 * reference's 1e-2 comparison rule (arke/agent/tools.py:510-517).  b per w_layout. */
ARKE_B200_API int arke_b200_matmul(const void* a, int64_t lda, const void* b, int64_t ldb, int w_layout,
                     int dtype, int64_t M, int64_t N, int64_t K, void* c, int64_t ldc,
                     void* stream);

/* C[M,N] = A^T B with A given as [K,M] (M contiguous, row stride lda) — the operand layout of a
 * weight-gradient GEMM (dW = G^T X).  16-bit operands (bf16 / f16), fp32 accumulate; B layout as in
 * arke_b200_matmul; c_dtype bf16 / f16 / f32.  The tensor core reads A as an "MN-major" shared-memory
 * operand, so no transposed copy of A is made. */
ARKE_B200_API int arke_b200_matmul_tn(const void* a, int64_t lda, const void* b, int64_t ldb, int w_layout,
                        int dtype, int64_t M, int64_t N, int64_t K, void* c, int c_dtype, int64_t ldc,
                        void* stream);

/* Causal / non-causal grouped-query flash-attention forward
 * (arke/ir/ops/reference_impls.py:236-244; arke/backend/triton_templates/flash_attention.py.j2).
 *   q [B,Hq,S,D], k,v [B,Hkv,Skv,D] contiguous bf16/f16, D = 128 or 64, Hq % Hkv == 0.
 *   o [B,Hq,S,D] same dtype; lse [B,Hq,S] fp32 natural-log logsumexp of the scaled, masked
 *   scores (may be NULL).  softmax_scale <= 0 selects 1/sqrt(D).  With causal != 0 query i sees
 *   keys j <= i (top-left aligned, as F.scaled_dot_product_attention(is_causal=True)). */
ARKE_B200_API int arke_b200_gqa_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int dtype,
                      int64_t B, int64_t Hq, int64_t Hkv, int64_t S, int64_t Skv, int64_t D,
                      int causal, float softmax_scale, void* stream);

/* Fused linear + cross-entropy without materialising logits
 * (arke/ir/ops/reference_impls.py:211-213): logits = X * W^T in fp32 from 16-bit inputs,
 * loss_i = logsumexp(logits_i) - logits_i[label_i], 0 for label_i == ignore_index.
 *   x [M,D], w [V,D] bf16/f16, labels [M] int64.
 *   loss_tok [M] fp32 (may be NULL), mean_loss [1] fp32 = sum / count(non-ignored) (may be NULL).
 *   partials [M,3] fp32 (may be NULL): per-row (max, sum exp(l - max), target logit or 0) over
 *   this call's vocabulary slice, for combining vocabulary shards; `vocab_offset` is the global
 *   index of w's first row (labels are global indices).
 *   A call with vocab_offset == 0 and partials == NULL covers the whole vocabulary for certain:
 *   a non-ignored label outside [0, V) (the reference's F.cross_entropy raises for it) then gives
 *   that row a NaN loss and records code 6 in the kernel status word.  Slice calls cannot tell a
 *   corrupt label from one that another slice holds and treat it as "not in this slice".
 *   workspace: at least arke_b200_fused_linear_ce_workspace(M, V, D) bytes of device memory. */
ARKE_B200_API size_t arke_b200_fused_linear_ce_workspace(int64_t M, int64_t V, int64_t D);
ARKE_B200_API int arke_b200_fused_linear_ce(const void* x, const void* w, const int64_t* labels, int dtype,
                              int64_t M, int64_t V, int64_t D, int64_t vocab_offset,
                              int64_t ignore_index, float* loss_tok, float* mean_loss,
                              float* partials, void* workspace, size_t workspace_bytes,
                              void* stream);

/* fused_linear_ce for hosts that cannot hand over a workspace.  No counterpart in the reference.
 * Same computation and arguments as arke_b200_fused_linear_ce, but the scratch memory is an 8 MiB
 * array built into the library (resident on every GPU that loads it until the process exits)
 * instead of a caller-allocated workspace: meant for callers whose device memory is entirely
 * owned by their own pool, or that must not trigger an allocation (and the device-wide stall it
 * can bring) where this op runs.  The call allocates and frees nothing.
 *   Limit: arke_b200_fused_linear_ce_workspace(M, V, D) must be <= 8 MiB (8388608 bytes), e.g.
 *   M <= 1024 tokens at V = 128256, or M <= 8192 at V <= 32000; larger problems are rejected with
 *   ARKE_ERR_WORKSPACE.
 *   The first call on each device resolves the array's device address: make it before any
 *   stream capture.  All calls share the array; calls that overlap on the GPU race on it, so
 *   order them on one stream (or with events). */
ARKE_B200_API int arke_b200_fused_linear_ce_static(const void* x, const void* w, const int64_t* labels, int dtype,
                                     int64_t M, int64_t V, int64_t D, int64_t vocab_offset,
                                     int64_t ignore_index, float* loss_tok, float* mean_loss,
                                     float* partials, void* stream);

/* Combines G vocabulary-shard partials [G,M,3] (layout above) into per-token loss and mean. */
ARKE_B200_API int arke_b200_ce_combine(const float* partials, int64_t G, int64_t M, const int64_t* labels,
                         int64_t ignore_index, float* loss_tok, float* mean_loss, void* stream);

/* Backward of fused linear + cross-entropy: gradients of the MEAN loss w.r.t. x and w.
 * The reference implements the forward only (arke/ir/ops/reference_impls.py:211-213); its operator
 * documentation promises a logits gradient (docs/benchmark/benchmark-ops.md:582-593) that none of
 * its backends produces.  Definition: with p = softmax(x w^T) per row and n = number of rows whose
 * label != ignore_index,
 *   G[i,j] = p[i,j] - [j == labels[i] - vocab_offset]                (rows with ignored label: 0)
 *   dx = (g / n) G w   [M,D],      dw = (g / n) G^T x   [V,D]        (fp32 accumulate)
 *   g = grad * (grad_dev ? *grad_dev : 1): `grad_dev` is an optional fp32 device scalar (the
 *   upstream gradient of a training step), so that no host read of it is needed.
 *   dx is written as `dx_dtype`: the operands' dtype, or ARKE_F32 (what a vocabulary-sharded
 *   caller sums over ranks without a 16-bit rounding per rank); dw has the operands' dtype.
 *   lse [M] fp32: natural-log logsumexp of each row's logits over the WHOLE vocabulary, as the
 *   forward's partials give it (max + log(sumexp)); with a vocabulary slice (vocab_offset, V rows
 *   of w) dx is this slice's contribution and the caller sums the slices' dx.
 *   dx / dw may be NULL (skipped).  workspace: arke_b200_fused_linear_ce_backward_workspace(M, V)
 *   bytes, 256-byte aligned (holds G, 16-bit and unscaled, [M, V rounded up to 8]). */
ARKE_B200_API size_t arke_b200_fused_linear_ce_backward_workspace(int64_t M, int64_t V);
ARKE_B200_API int arke_b200_fused_linear_ce_backward(const void* x, const void* w, const int64_t* labels,
                                       const float* lse, int dtype, int64_t M, int64_t V, int64_t D,
                                       int64_t vocab_offset, int64_t ignore_index, float grad,
                                       const float* grad_dev, void* dx, int dx_dtype, void* dw,
                                       void* workspace, size_t workspace_bytes, void* stream);

/* A ragged batch over a paged key/value cache (bf16 / f16).  The reference has no cache: its
 * attention ops read whole sequences (arke/ir/ops/reference_impls.py:236-244).
 *   k, v       row p % page_size of page block_table[b][p / page_size] holds position p of sequence
 *              b; element (page, head, row, d) is at page * stride_page + head * stride_head +
 *              row * stride_row + d, so head-major, token-major and interleaved buffers all fit;
 *   block_table [batch, max_pages] int32, row stride ld_table; entries behind a sequence's last page
 *              are never read;
 *   kv_lens    [batch] int32: positions of each sequence, the new tokens of this call included;
 *   cu_q       [batch + 1] int32, non-decreasing from 0: sequence b owns the query rows
 *              [cu_q[b], cu_q[b + 1]); NULL: T / batch rows each.  Rows from cu_q[batch] to T belong to
 *              no sequence: their outputs are zero.  The tokens of a sequence are its last ones:
 *              row i of n has position kv_lens[b] - n + i;
 *   max_new    no less than the longest sequence's query rows, or 0 if unknown.  Only paged_gqa_fwd's choice of
 *              kernels goes by it, and only with cu_q: results are right whatever it says.  Unknown, every
 *              sequence is taken to have a row, which a batch of mostly empty slots pays for.
 * A page outside [0, num_pages), a length below 0 or beyond max_pages * page_size, or (append) a
 * position below 0 or outside the cos / sin tables sets status code 8; nothing is read or written there. */
typedef struct {
  void* k;
  void* v;
  int64_t k_stride_page, k_stride_head, k_stride_row;
  int64_t v_stride_page, v_stride_head, v_stride_row;
  int64_t num_pages, page_size, heads, head_dim;
  const int32_t* block_table;
  int64_t ld_table, max_pages;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  int64_t batch;
  int32_t dtype;
  int32_t max_new;
} arke_b200_paged_kv;

/* qkv_rope_split for a paged cache: qkv [T, ld] holds, per token, Hq query heads, then the key heads,
 * then the value heads.  Queries and keys are rotated (rotate-half form, as arke_b200_rope) in fp32 and
 * rounded once; q [T, Hq, D] contiguous; keys and values are written to their pages, everything else
 * in the cache is left as it was.  Two sequences must not own the page a new token goes to, and the
 * cache must not be an expanded view (a stride of 0).
 *   cos, sin [table_rows, D/2] contiguous, f32 or the cache's type; row = the token's position, or
 *   positions[t] (int32 [T]) where it is given.  D even.
 * A token whose page or table row does not exist is not stored (status code 8); its q is NaN when the
 * table row is missing. */
ARKE_B200_API int arke_b200_qkv_rope_paged_append(const void* qkv, int64_t ld, const void* cos, const void* sin,
                                    int table_dtype, int64_t table_rows, const int32_t* positions,
                                    const arke_b200_paged_kv* kv, void* q, int64_t T, int64_t Hq,
                                    void* stream);

/* Grouped-query attention of a ragged batch over a paged cache: row i of n of sequence b (L positions)
 * sees positions j <= L - n + i (causal != 0, aligned to the sequence's end) or all L.
 *   q [T, Hq, D] with strides (token, head), D contiguous, 64 or 128; o [T, Hq, D] contiguous, type of
 *   q and the cache; lse [T, Hq] fp32 natural-log logsumexp (may be NULL).  A row that sees nothing:
 *   o = 0, lse = -inf.  softmax_scale <= 0 selects 1/sqrt(D).  A key that a row does not see may hold
 *   anything; so may memory behind a sequence's end.  A NaN or infinity among the values of a sequence's
 *   own positions can reach its rows that do not see that position (a weight of 0 times it is NaN), in a shared
 *   prefix rows of every sequence.
 *   shared_prefix: the first positions [0, shared_prefix) of every sequence are the same (of a shorter one,
 *   all that it has; behind the longest sequence nothing is read).  Their whole
 *   pages are read through sequence 0's row of the block table, and once for the whole batch where that
 *   pays; of a page that the prefix fills in part every sequence has its own.  0 = nothing shared.
 *   A page outside its range: the rows that see one of its positions are NaN, o and lse, and other rows of that
 *   sequence may be (of the batch, when it lies in the shared prefix).  A length outside its range: every row of
 *   that sequence is NaN.  Both set status code 8.
 *   Accuracy: scores, sums and partial results are fp32.  The weights meet the values with 17 bits or more; where many
 *   rows read the same keys (more than 32 rows times heads per key head of a sequence, or a prefix computed apart) they
 *   are rounded to the cache's type first, which moves a result by half a step of sum_j p_j |v_j| at most.
 *   workspace: arke_b200_paged_gqa_workspace(...) bytes, 256-byte aligned; contents need no
 *   initialisation and nothing is kept in it between calls; calls that may overlap need one each. */
ARKE_B200_API size_t arke_b200_paged_gqa_workspace(int64_t T, int64_t batch, int64_t Hq, int64_t Hkv, int64_t D,
                                     int64_t shared_prefix);
ARKE_B200_API int arke_b200_paged_gqa_fwd(const void* q, int64_t q_stride_token, int64_t q_stride_head,
                            const arke_b200_paged_kv* kv, void* o, float* lse, int64_t T, int64_t Hq,
                            int64_t shared_prefix, int causal, float softmax_scale, void* workspace,
                            size_t workspace_bytes, void* stream);

/* Chooses one token per row of logits [B, V] (bf16 / f16 / f32, row stride ld, V <= 2^20) with a given random number
 * u[row] in [0, 1).  The reference has no sampler.  With w_i = exp((x_i - max x) / temperature), the
 * tokens ranked by x, equal values by their index:
 *   top_k  keeps the first k (0, or k >= V: all);
 *   top_p  keeps those of them whose predecessors weigh less than top_p times what top_k kept (>= 1:
 *          all; the first is always kept);
 *   min_p  keeps w_i >= min_p (0: all);
 *   token  = the first kept index i, in vocabulary order, with sum_{j <= i, kept} w_j > u * Z, Z the sum
 *            of what is kept;  logprob [B] (may be NULL) = log(w_token / Z), rounded once; in rows that
 *            neither top_k nor top_p cuts, Z may be a sum of single-precision weights, and logprob off by up to 2^-17.
 * temperature <= 0: the arg max (lowest index), logprob 0.  A NaN logit counts as -inf, which is never
 * chosen; a row of -inf alone gives token -1, logprob -inf.  u outside [0, 1) is clamped; at u = 0 the first
 * kept token whose weight is not zero in 64 bits is chosen.  Decisions are those of 64-bit arithmetic and do not
 * depend on how the work is split: a weight is off by 2^-42 of itself and 2^-85 of the largest, where top_p
 * looks for its border by 2^-60 of the largest.
 * A value for all rows must be in range (temperature, top_k, top_p >= 0, min_p in [0, 1]); of arrays, negative entries
 * count as 0.  Each parameter is a value for all rows, or a device array [B] (fp32; top_k int32) where it is not NULL. */
ARKE_B200_API int arke_b200_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t B, int64_t V,
                            const float* u, const float* temperature_row, float temperature,
                            const int32_t* top_k_row, int64_t top_k, const float* top_p_row, float top_p,
                            const float* min_p_row, float min_p, int64_t* token, float* logprob,
                            void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ARKE_B200_H */
