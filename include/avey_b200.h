/*
 * avey_b200.h -- C ABI of the B200 (sm_100a) contextualizer forward library.
 *
 * One call computes, for every batch row b,
 *
 *   out[b] = z_tl[b] * act( (S_b (.) V (.) M_b) z_tr[b] / den_b + bias )
 *
 * with S_b the cosine similarity of the rows of z_tr[b], M_b the causal and
 * padding mask and den_b the signed row sum (Avey-B) or 1 (Avey): the math of
 * the reference's avey_kernels/ops.py:61-91 (_reference).
 *
 * The library is plain C at this boundary: raw device pointers, element
 * strides and sizes, no framework types. It never throws; every entry point
 * returns an AveyStatus and avey_last_error() describes the last failure on
 * the calling thread. Calls only enqueue work on the given stream: they do not
 * synchronise and do not allocate (scratch memory, when a kernel needs it, is
 * passed in by the caller as `workspace`), so they can be captured in a CUDA
 * graph.
 */
#ifndef AVEY_B200_H
#define AVEY_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AVEY_ABI_VERSION 5

#if defined(__GNUC__)
#define AVEY_API __attribute__((visibility("default")))
#else
#define AVEY_API
#endif

/* Element types of z_tr, v, z_tl, bias and out (all share one type). */
typedef enum AveyDtype {
  AVEY_F32 = 0,
  AVEY_F16 = 1,
  AVEY_BF16 = 2,
  AVEY_F64 = 3,
} AveyDtype;

/* Activation ids; the numbering is that of the reference, _triton.py:169. */
typedef enum AveyActivation {
  AVEY_ACT_IDENTITY = 0,
  AVEY_ACT_RELU = 1,
  AVEY_ACT_RELU2 = 2,
  AVEY_ACT_SILU = 3,
  AVEY_ACT_GELU = 4, /* tanh approximation */
} AveyActivation;

/* Kernel selection. AUTO picks the tcgen05 kernels whenever the shape, dtype
 * and alignment allow it, except for small fp32 problems (contexts up to
 * 512, features a multiple of 32 up to 256, a few waves of 8-row query
 * tiles), which finish sooner on an 8-row CUDA-core kernel (AveyPlan.reason
 * 6); else the general CUDA-core kernel. AVEY_KERNEL_SIMT forces the general
 * CUDA-core kernel, AVEY_KERNEL_TCGEN05 the tcgen05 kernels. */
typedef enum AveyKernel {
  AVEY_KERNEL_AUTO = 0,
  AVEY_KERNEL_SIMT = 1,   /* general CUDA-core kernel: any dtype/stride/shape */
  AVEY_KERNEL_TCGEN05 = 2 /* TMA + tcgen05 + TMEM kernels (bf16 / f16): one fused
                             kernel up to 512 tokens, two kernels from 513 to 8192 */
} AveyKernel;

typedef enum AveyStatus {
  AVEY_OK = 0,
  AVEY_ERR_ARGUMENT = -1,    /* bad size, pointer, stride, flag or struct */
  AVEY_ERR_ARCH = -2,        /* current device is not sm_100 */
  AVEY_ERR_UNSUPPORTED = -3, /* a forced kernel cannot run these inputs */
  AVEY_ERR_LAUNCH = -4,      /* the CUDA launch itself failed */
  AVEY_ERR_DEVICE = -5,      /* a kernel reported a timeout or fault flag */
  AVEY_ERR_CUDA = -6,        /* another CUDA runtime / driver call failed */
} AveyStatus;

/*
 * Forward parameters. Strides are in ELEMENTS. The feature (last) dimension
 * of z_tr, z_tl and out must have stride 1; the other strides are free, so the
 * head and tail halves of one [B, C, 2d'] tensor are passed as two views
 * (row stride 2d') without a copy. Optional tensors are NULL when absent.
 * valid holds one byte per (batch, position): nonzero = valid.
 */
typedef struct AveyFwdParams {
  uint32_t struct_size; /* sizeof(AveyFwdParams); guards ABI drift */
  int32_t dtype;        /* AveyDtype */
  int64_t batch;        /* B  >= 1 */
  int64_t context;      /* C  >= 1 (tokens per batch row) */
  int64_t features;     /* d' >= 1 */

  const void* z_tr;     /* [B, C, d'] tail half (required) */
  int64_t z_tr_batch_stride, z_tr_row_stride;
  const void* v;        /* [C, C] indexed [query, key] (Avey) or NULL */
  int64_t v_row_stride;
  const void* z_tl;     /* [B, C, d'] head half, the gate, or NULL */
  int64_t z_tl_batch_stride, z_tl_row_stride;
  const void* bias;     /* [d'] contiguous, or NULL */
  const uint8_t* valid; /* [B, C] bytes, or NULL */
  int64_t valid_batch_stride, valid_row_stride;
  void* out;            /* [B, C, d'] output, same dtype as z_tr */
  int64_t out_batch_stride, out_row_stride;

  double eps;      /* Avey-B denominator epsilon (used when normalize != 0) */
  double norm_eps; /* L2-normalisation epsilon: x / max(||x||, norm_eps) */
  int32_t causal;     /* keep key j <= query i (diagonal kept) */
  int32_t normalize;  /* divide by the signed row sum + eps (Avey-B) */
  int32_t activation; /* AveyActivation */
  int32_t kernel;     /* AveyKernel */
  void* workspace;          /* device scratch, >= avey_fwd_workspace_size() bytes */
  uint64_t workspace_bytes; /* size of `workspace` in bytes */

  /* Prefix form of the padding mask, instead of `valid` (passing both is an
   * error): a device array of B int32 lengths, positions [0, lengths[b]) of
   * batch row b are valid and the rest is padding (values above the context
   * act as the context, values below 1 leave the row all padding). No mask
   * bytes are read. The reference takes only the byte mask (ops.py:23-46);
   * this is the C-ABI fast path for callers that hold lengths. */
  const int32_t* lengths;
} AveyFwdParams;

/* What avey_fwd_v1 would launch for these parameters. */
typedef struct AveyPlan {
  int32_t kernel;        /* AVEY_KERNEL_SIMT or AVEY_KERNEL_TCGEN05 */
  int32_t launches;      /* kernel launches per call: 1 on the tcgen05 path up to
                            512 tokens (the fused kernel), 3 above (row-sum pre-pass,
                            G/P kernel, O = P Z kernel), 2 for fp32 on the 3xTF32
                            pair, 1 on CUDA cores */
  int32_t grid;          /* CTAs of the main launch */
  int32_t block;         /* threads per CTA of the main launch */
  int32_t smem_bytes;    /* dynamic shared memory per CTA */
  int32_t reason;        /* 0, or why the tcgen05 kernel was not chosen: 1 dtype,
                            2 context, 3 alignment, 4 AVEY_KERNEL_SIMT asked for,
                            5 features, 6 small fp32 problem (AUTO runs the 8-row
                            CUDA-core kernel, which finishes first there) */
} AveyPlan;

/*
 * Run the contextualizer forward on `stream` (a cudaStream_t; NULL is the
 * legacy default stream). Replaces, in the reference, the normalisation
 * pre-pass plus the fused mixing launch: avey_kernels/ops.py:107-114
 * (F.normalize into a temporary fp32 buffer, then mix) and
 * avey_kernels/_triton.py:153-188 (the avey_kernels::mix custom op that
 * launches _mix_kernel). Normalisation is fused into the kernel here.
 * Returns AVEY_OK or a negative AveyStatus.
 */
AVEY_API int avey_fwd_v1(const AveyFwdParams* params, void* stream);

/* Fill *plan with the launch avey_fwd_v1 would make; launches nothing.
 * Has no reference counterpart (introspection for tests and benchmarks). */
AVEY_API int avey_fwd_plan(const AveyFwdParams* params, AveyPlan* plan);

/* Device workspace avey_fwd_v1 needs for these parameters, in bytes: 0 for the
 * CUDA-core kernels and for the fused tcgen05 kernel (up to 512 tokens: it
 * sums the rows' squares from the tiles it stages); above 512 tokens and for
 * fp32 on the 3xTF32 pair, in 256-byte aligned parts, the row sums of squares
 * (4 bytes per row of z_tr), 4 bytes per row per group of 256 keys (partial
 * row sums) and P itself (2 bytes per (query, key) pair, 4 for fp32, rows
 * padded to 64 keys): 134 MB for batch 16 x 2048 tokens. The workspace must
 * be 256-byte aligned. The reference allocates its normalisation buffer
 * itself (ops.py:108); this library leaves allocation to the caller.
 * Launches nothing. */
AVEY_API int avey_fwd_workspace_size(const AveyFwdParams* params, uint64_t* bytes);

/*
 * avey_fwd_v1 for callers that cannot allocate device memory: no counterpart
 * in the reference. Some callers hold no device allocator of their own -- an
 * FFI host (cgo, JNI, a plugin ABI) that only passes raw pointers in, or code
 * that runs while a stream is being captured into a CUDA graph, where
 * allocation is not allowed -- so they cannot provide `workspace`. This entry
 * point ignores params->workspace and uses a scratch array that lives inside
 * the library instead (file-scope device memory, present on every GPU that
 * loads the library until the process exits). It allocates nothing.
 *
 * Contexts above 512 tokens run the CUDA-core kernel here (the tcgen05 path
 * for them needs a P workspace); forcing AVEY_KERNEL_TCGEN05 for them fails
 * with AVEY_ERR_UNSUPPORTED.
 *
 * On the fused tensor-core path (bf16 / f16 up to 512 tokens) this entry point
 * runs the kernel's pre-pass variant: a row-norm pre-pass writes each row's
 * sum of squares into the array and the fused kernel reads them, where
 * avey_fwd_v1 has the fused kernel sum the rows itself; the two agree to
 * the rounding of those sums.
 *
 * Limit: on the fused tensor-core path (the only path that reads the
 * scratch) batch * context <= AVEY_NOALLOC_MAX_ROWS
 * (1,048,576 rows; the array holds one float per row, 4 MiB per GPU); larger
 * inputs are rejected with AVEY_ERR_ARGUMENT. Inputs that run a CUDA-core
 * kernel use no scratch and have no such limit. The first call on each device
 * looks up the array's
 * device address (with that device current); make that first call before
 * any stream capture. All calls share the one array, so calls whose kernels
 * overlap on the GPU (for example on two streams) race; each call rewrites
 * every row it reads, so nothing needs clearing between calls.
 */
#define AVEY_NOALLOC_MAX_ROWS (1u << 20)
AVEY_API int avey_fwd_noalloc_v1(const AveyFwdParams* params, void* stream);

/*
 * Backward pass. The reference has no fused backward: autograd runs through
 * its PyTorch path (avey_kernels/ops.py:94-106 send any input that requires
 * grad to _reference, ops.py:61-91). This library splits the gradient into
 * five batched GEMMs, which the caller runs with a library GEMM, and five
 * fused steps that run here between them:
 *
 *   AVEY_BWD_PREP      zm = z_tr (padded rows 0), norms = ||zm|| (-1: padding)
 *                                                          then  g = zm zm^T
 *   AVEY_BWD_SCORES    s = g r_i r_j (.) v (.) mask, den = rowsum(s) + eps,
 *                      r = 1 / max(norms, norm_eps)        then  num = s zm
 *   AVEY_BWD_EPILOGUE  grad_z_tl, grad_bias, dnum, dden from grad_out
 *                                        then  ds0 = dnum zm^T, dzd = s^T dnum
 *   AVEY_BWD_DSCORES   dgsym = (dG + dG^T) diag(r), dG = (ds0 + dden) (.)
 *                      mask (.) v; grad_v                  then  dzh = dgsym zm
 *   AVEY_BWD_FINAL     grad_z_tr = dzd + normalisation backward of dzh
 *
 * GEMM operands (zm, s, dnum, dgsym) are of gemm_dtype: AVEY_BF16 for
 * bf16 inputs, AVEY_F32 for f16 and f32 inputs, AVEY_F64 for f64 inputs.
 * Accumulator arrays (norms, g, den, num, dden, ds0, dzd, dzh, workspace) are
 * float, or double for f64 inputs; GEMM outputs are written in that type. All
 * scratch arrays are contiguous ([B, C, d'], [B, C, C] or [B, C]); the
 * gradients are of the input dtype, and an output pointer left NULL is not
 * computed (grad_v needs v, grad_z_tl needs z_tl). Reductions use
 * fixed orders: results are bitwise reproducible.
 */
typedef enum AveyBwdStep {
  AVEY_BWD_PREP = 0,
  AVEY_BWD_SCORES = 1,
  AVEY_BWD_EPILOGUE = 2,
  AVEY_BWD_DSCORES = 3,
  AVEY_BWD_FINAL = 4,
} AveyBwdStep;

typedef struct AveyBwdParams {
  uint32_t struct_size; /* sizeof(AveyBwdParams) */
  int32_t dtype;        /* AveyDtype of the inputs and gradients */
  int32_t gemm_dtype;   /* AveyDtype of the GEMM operand arrays (see above) */
  int32_t causal, normalize, activation;
  int64_t batch, context, features;
  double eps, norm_eps;

  /* Forward inputs, strided as in AveyFwdParams. */
  const void* z_tr;
  int64_t z_tr_batch_stride, z_tr_row_stride;
  const void* v;
  int64_t v_row_stride;
  const void* z_tl;
  int64_t z_tl_batch_stride, z_tl_row_stride;
  const void* bias;
  const uint8_t* valid;
  int64_t valid_batch_stride, valid_row_stride;
  const void* grad_out; /* [B, C, d'] gradient of the forward output */
  int64_t grad_out_batch_stride, grad_out_row_stride;

  /* Scratch written by one step and read by later ones or by the GEMMs. */
  void* zm;        /* [B, C, d'] gemm_dtype; may be NULL when valid is NULL and
                      gemm_dtype == dtype (zm would equal z_tr): PREP then writes
                      only the norms, FINAL reads z_tr, and the caller's GEMMs
                      take z_tr (strided) in place of zm */
  void* norms;     /* [B, C]     acc: ||zm||, -1 on padded positions */
  void* g;         /* [B, C, C]  acc (GEMM output) */
  void* s;         /* [B, C, C]  gemm_dtype */
  void* den;       /* [B, C]     acc */
  void* num;       /* [B, C, d'] acc (GEMM output) */
  void* dnum;      /* [B, C, d'] gemm_dtype */
  void* dden;      /* [B, C]     acc */
  void* ds0;       /* [B, C, C]  acc (GEMM output) */
  void* dgsym;     /* [B, C, C]  gemm_dtype */
  void* dzd;       /* [B, C, d'] acc (GEMM output) */
  void* dzh;       /* [B, C, d'] acc (GEMM output) */
  void* workspace; /* partial sums, >= avey_bwd_workspace_size() bytes */
  uint64_t workspace_bytes;

  /* Gradients (input dtype); NULL = not wanted. grad_v and grad_bias are
   * contiguous; grad_z_tr and grad_z_tl share the element strides below
   * (0 = contiguous [B, C, d']), so both can be the halves of one
   * [B, C, 2d'] gradient (row stride 2d'). */
  void* grad_z_tr;
  void* grad_v;
  void* grad_z_tl;
  void* grad_bias;
  int64_t grad_batch_stride, grad_row_stride;
} AveyBwdParams;

/* Enqueue one backward step on `stream`. Returns AVEY_OK or a negative
 * AveyStatus; the pointers a step reads or writes must be set. */
AVEY_API int avey_bwd_step_v1(const AveyBwdParams* params, int step, void* stream);

/*
 * Batched matrix product on the tcgen05 tensor cores (no counterpart in the
 * reference, which computes its products with torch.matmul / tl.dot): for
 * every batch entry b,
 *
 *   C[b] = A[b] B[b]                              out_dtype AVEY_F32, or
 *   C[b] = act(A[b] B[b] + bias) (.) gate[b]      out_dtype == dtype (16-bit)
 *
 * with A [m x k] and B [k x n] of `dtype` (AVEY_BF16 or AVEY_F16) and fp32
 * accumulation. It runs the contractions of the backward steps above
 * (avey_kernel_b200/backward.py), the enricher projection that feeds
 * avey_fwd_v1 (with the row sums of squares of its tail columns, see
 * avey_fwd_presummed_v1) and the static layers.
 *
 * Layouts (strides in elements, each operand's contiguous dimension has
 * stride 1):
 *   A: a_major AVEY_MAJOR_K:  A[b][i][k] at a + b*a_batch_stride + i*a_ld + k
 *      a_major AVEY_MAJOR_MN: A[b][i][k] at a + b*a_batch_stride + k*a_ld + i
 *   B: b_major AVEY_MAJOR_K:  B[b][k][j] at b + b*b_batch_stride + j*b_ld + k
 *      b_major AVEY_MAJOR_MN: B[b][k][j] at b + b*b_batch_stride + k*b_ld + j
 *   C: C[b][i][j] at c + b*c_batch_stride + i*c_ld + j
 * A batch stride of 0 shares the operand across the batch. Base addresses
 * must be 16-byte aligned and every ld / batch stride a whole number of 16
 * bytes (TMA); k, m and n are otherwise free (edges are zero-filled).
 *
 * mode skips work that the causal structure makes unnecessary:
 *   AVEY_GEMM_DENSE      every C[b][i][j];
 *   AVEY_GEMM_LOWER_OUT  only C[b][i][j] with j <= i is wanted: 128 x 256
 *                        output tiles wholly above the diagonal are not
 *                        computed and not written (their memory keeps
 *                        whatever it held);
 *   AVEY_GEMM_K_LOWER    A[b][i][k] == 0 for k > i (lower-triangular A): the
 *                        K loop of each 128-row tile stops after its last row;
 *   AVEY_GEMM_K_UPPER    A[b][i][k] == 0 for k < i: the K loop of each
 *                        128-row tile starts at its first row.
 * The K-range modes give the dense result bit for bit (the skipped terms are
 * exact zeros).
 *
 * 16-bit output only: bias [n] (or NULL), activation (AveyActivation), gate
 * (same shape as C, or NULL), and sumsq: NULL, or n_planes = ceil((n -
 * sumsq_col0) / 128) planes of batch*m floats, plane p holding for every row
 * the sum of squares of the stored (rounded) outputs of columns
 * [sumsq_col0 + 128p, sumsq_col0 + 128p + 128) (sumsq_col0 a multiple of 128;
 * sums in a fixed order, bitwise reproducible).
 */
typedef enum AveyMajor {
  AVEY_MAJOR_K = 0,
  AVEY_MAJOR_MN = 1,
} AveyMajor;

typedef enum AveyGemmMode {
  AVEY_GEMM_DENSE = 0,
  AVEY_GEMM_LOWER_OUT = 1,
  AVEY_GEMM_K_LOWER = 2,
  AVEY_GEMM_K_UPPER = 3,
} AveyGemmMode;

typedef struct AveyGemmParams {
  uint32_t struct_size; /* sizeof(AveyGemmParams) */
  int32_t dtype;        /* operands: AVEY_BF16 or AVEY_F16 */
  int32_t out_dtype;    /* AVEY_F32, or dtype */
  int32_t mode;         /* AveyGemmMode */
  int64_t batch, m, n, k;
  const void* a;
  int64_t a_batch_stride, a_ld;
  int32_t a_major; /* AveyMajor */
  const void* b;
  int64_t b_batch_stride, b_ld;
  int32_t b_major; /* AveyMajor */
  void* c;
  int64_t c_batch_stride, c_ld;
  const void* bias; /* [n] of dtype, or NULL (16-bit output only) */
  const void* gate; /* [batch][m][n] of dtype, or NULL (16-bit output only) */
  int64_t gate_batch_stride, gate_ld;
  int32_t activation; /* AveyActivation (16-bit output only) */
  int32_t sumsq_col0; /* first column of the row sums of squares */
  float* sumsq;       /* planes of row sums of squares, or NULL */
  int32_t kernel;     /* AVEY_GEMM_KERNEL_*: AUTO runs SINGLE (measured the
                         faster of the two on every shape tried) */
} AveyGemmParams;

/* GEMM kernels: one CTA per 128 x 256 output tile, or a pair of CTAs on
 * neighbouring SMs per 256 x 256 tile sharing each MMA (tcgen05 cta_group::2),
 * which halves the B bytes each SM loads per MMA cycle. Same results. */
#define AVEY_GEMM_KERNEL_AUTO 0
#define AVEY_GEMM_KERNEL_SINGLE 1
#define AVEY_GEMM_KERNEL_PAIR 2

AVEY_API int avey_gemm_v1(const AveyGemmParams* params, void* stream);

/*
 * avey_fwd_v1 with the row sums of squares of z_tr supplied by the caller
 * (no counterpart in the reference, whose normalisation pre-pass,
 * ops.py:107-108, is always a separate pass over z_tr): `sumsq` holds
 * `planes` planes of batch*context floats, summed in plane order, as written
 * by the enricher's avey_gemm_v1 epilogue (its tail columns). The norm
 * fused tcgen05 kernel and the long-context path read these sums instead of
 * summing z_tr's rows; other paths ignore them. Up to 512 tokens the planes
 * are combined into params->workspace, which must then hold batch * context
 * floats (4-byte aligned); above 512 tokens the workspace is the one
 * avey_fwd_workspace_size reports.
 */
AVEY_API int avey_fwd_presummed_v1(const AveyFwdParams* params, const float* sumsq, int planes,
                                   void* stream);

/*
 * Linear layers with a fused epilogue, dense or grouped by expert, and their
 * gradients (no counterpart in the reference, which leaves the layers around
 * the contextualizer to torch.matmul):
 *
 *   forward   y  = act(x W_g^T + b_g) + residual
 *   backward  dpre = dy (.) act'(x W_g^T + b_g)
 *             dx = dpre W_g, dweight_g = dpre_g^T x_g, dbias_g = sum of dpre_g
 *             (the residual's gradient is dy itself)
 *
 * on x [rows][d_in], W [groups][d_out][d_in], b [groups][d_out]. With offsets
 * (device, groups + 1 values) group g owns the rows [offsets[g], offsets[g +
 * 1]); offsets[0] is taken as 0, values out of order or out of range are pulled
 * into [the group's start, rows], and rows from offsets[groups] on belong to no
 * group: their y and dx are zero and they add to no gradient. Without offsets
 * (groups == 1) every row belongs to the one group. Group sizes are never read
 * back to the host.
 *
 * dtype is AVEY_BF16 or AVEY_F16 for every array; products and sums are fp32
 * and each result is rounded once; dpre is rounded to dtype before the two
 * products of the backward pass. The forward pass writes act' as 16-bit codes
 * into deriv when it is given (d_out rounded up to 16 values a row; any
 * activation but the identity), and the backward pass reads them: relu exactly,
 * silu and gelu to 2^-15, relu2 to 2^-10 of itself from 2^-62 to 2^66 (bf16) or
 * 2^-12 from 2^-15 to 2^10 (f16) and as 0 below, so wherever y is finite. Gradients
 * use fixed orders: results are bitwise reproducible.
 *
 * Last dimensions have stride 1; row strides (ld) and group strides are in
 * elements. Any alignment is taken: rows that are not whole 16-byte units
 * are copied into the workspace first where the tensor cores read them.
 */
typedef struct AveyLinearParams {
  uint32_t struct_size; /* sizeof(AveyLinearParams) */
  int32_t dtype;        /* AVEY_BF16 or AVEY_F16 */
  int32_t activation;   /* AveyActivation */
  int32_t kernel;       /* AVEY_LINEAR_KERNEL_* (forward) */
  int64_t rows, d_in, d_out, groups; /* up to 2^30, 2^22, 2^22 and 65535 */
  const int32_t* offsets;
  const void* x;
  int64_t x_ld;
  const void* weight;
  int64_t weight_ld, weight_group_stride;
  const void* bias; /* or NULL */
  int64_t bias_group_stride;
  const void* residual; /* [rows][d_out], or NULL */
  int64_t residual_ld;
  void* y;
  int64_t y_ld;
  void* deriv; /* 32-byte aligned; forward: or NULL */

  /* Backward (y, residual and bias are not read, x for dweight only and weight
   * for dx only). NULL: not wanted. */
  const void* dy; /* [rows][d_out] */
  int64_t dy_ld;
  void* dx; /* [rows][d_in] */
  int64_t dx_ld;
  void* dweight; /* contiguous [groups][d_out][d_in] */
  void* dbias;   /* contiguous [groups][d_out] */

  void* workspace; /* 256-byte aligned, >= avey_linear_workspace_size() bytes */
  uint64_t workspace_bytes;
} AveyLinearParams;

/* AUTO: the kernel for few rows, which reads the weights without filling
 * 128-row tiles, up to 8 rows, up to 256 by the size of the product (2^28
 * multiplications and about), and up to 64 grouped ones (by the size too where a
 * group has more than 8 rows on average); tcgen05 tiles above. */
#define AVEY_LINEAR_KERNEL_AUTO 0
#define AVEY_LINEAR_KERNEL_TCGEN05 1
#define AVEY_LINEAR_KERNEL_FEW 2

AVEY_API int avey_linear_fwd_v1(const AveyLinearParams* params, void* stream);
AVEY_API int avey_linear_bwd_v1(const AveyLinearParams* params, void* stream);

/* Bytes of `workspace` of the forward (backward == 0) or backward call. */
AVEY_API int avey_linear_workspace_size(const AveyLinearParams* params, int backward, uint64_t* bytes);

/*
 * Softmax cross entropy of z = x W^T over a vocabulary, without keeping z, and
 * its gradients (no counterpart in the reference, which leaves the loss to
 * torch). For row i with the target t_i:
 *
 *   lse_i  = log sum_j exp(z_ij)
 *   loss_i = lse_i - z_{i,t_i} + z_loss lse_i^2, or 0 where t_i = ignore_index
 *   loss   = loss_i (NONE), their sum (SUM), or the sum over the number of rows
 *            that are not ignored (MEAN; of none: NaN)
 *
 * on x [rows][width] and W [vocab][width]. A target outside [0, vocab) that is not
 * ignore_index makes its row's loss, and what depends on it, NaN. Ignored rows
 * have no part in anything, whatever x holds there, and their dx is zero.
 *
 * The forward call writes `saved` (rows + 1 floats: lse_i / log 2, and the bits of
 * the number of rows that count) and `saved_low` (what fp32 leaves out of lse_i / log 2)
 * for the backward call, which computes z again in pieces of the vocabulary, from dloss
 * (rows values dloss_stride apart for NONE, else one). Without `saved_low`, p - 1 of a row
 * that is sure of its target is off by 2^-24 |lse|.
 *
 *   dz_ij = g_i ((1 + 2 z_loss lse_i) exp(z_ij - lse_i) - [j = t_i])
 *   dx = dz W, dweight = dz^T x
 *
 * Products and sums are fp32; dz is rounded to dtype before its products (divided by the
 * largest |g_i| and scaled by a power of two, so that f16 does not lose small
 * probabilities) and each result once. Sums are taken in fixed orders: results are bitwise reproducible.
 *
 * Last dimensions have stride 1; x_ld, weight_ld, dx_ld and target_stride are in
 * elements (target_stride >= 0). Any alignment is taken: rows that are not whole
 * 16-byte units are copied into the workspace first.
 */
#define AVEY_LOSS_NONE 0
#define AVEY_LOSS_SUM 1
#define AVEY_LOSS_MEAN 2

typedef struct AveyLossParams {
  uint32_t struct_size; /* sizeof(AveyLossParams) */
  int32_t dtype;        /* AVEY_BF16 or AVEY_F16: x, weight, dx, dweight */
  int32_t target_bits;  /* 32 or 64: signed targets */
  int32_t reduction;    /* AVEY_LOSS_* */
  int64_t rows, width, vocab; /* up to 2^30, 2^22 and 2^30 */
  const void* x;
  int64_t x_ld;
  const void* weight;
  int64_t weight_ld;
  const void* targets;
  int64_t target_stride;
  int64_t ignore_index;
  double z_loss;
  float* loss;  /* forward: [rows] (NONE) or one value */
  float* saved; /* [rows + 1]; forward: or NULL */

  /* Backward. NULL: not wanted. */
  const float* dloss;
  int64_t dloss_stride;
  void* dx;
  int64_t dx_ld;
  void* dweight; /* contiguous [vocab][width] */

  void* workspace; /* 256-byte aligned, >= avey_loss_workspace_size() bytes */
  uint64_t workspace_bytes;
  float* saved_low; /* [rows], or NULL in both calls (or a block that ends before it) */
} AveyLossParams;

AVEY_API int avey_loss_fwd_v1(const AveyLossParams* params, void* stream);
AVEY_API int avey_loss_bwd_v1(const AveyLossParams* params, void* stream);

/* Bytes of `workspace` of the forward (backward == 0) or backward call, at most:
 *   backward: 512 MB for pieces of dz, or 16 KB a row above 32768 rows, and 1 KB a row to make them
 *     whole tiles; 6 bytes for every element of x, its rows filled up to 8; 32 bytes a row; and for
 *     the sums of dx's tiles that CTAs share 512 KB for each SM (without dweight 2 MB);
 *   forward: the larger of 5 MB and 8 bytes a row for every 1024 words, and 8 bytes a row;
 *   either: where the rows of x, or of the weight, are not whole 16-byte units (address, stride or
 *     width), a copy of that array, 2 bytes an element, its rows filled up to 8. */
AVEY_API int avey_loss_workspace_size(const AveyLossParams* params, int backward, uint64_t* bytes);

/*
 * Routing of tokens to experts (no counterpart in the reference). For each token, with z
 * its logits:
 *
 *   s = softmax(z) or sigmoid(z);   rank = z without a bias, else s + bias
 *   a group of experts / groups consecutive experts ranks by the sum of the ranks of its
 *   best group_best experts (1 or 2; without a bias by z for 1, by s for 2), and the
 *   experts of the best top_groups groups are chosen from
 *   chosen = the k of them that rank best, from the best on
 *   weights = scale s, or with renormalize scale s / (sum of s over the chosen)
 *
 * Ties go to the lowest index. The order is that of the formula in exact arithmetic:
 * where ranks in fp32 are too near to tell they are computed again in 64 bits. A logit
 * of -inf ranks its expert below every other, whatever its bias, and gives the weight 0
 * (also where all are -inf); a NaN ranks last and makes the softmax, or its own
 * sigmoid, NaN. The weights' gradient goes to the logits; the choice and the bias have none.
 */
#define AVEY_SCORE_SOFTMAX 0
#define AVEY_SCORE_SIGMOID 1

typedef struct AveyRouteParams {
  uint32_t struct_size; /* sizeof(AveyRouteParams) */
  int32_t dtype;        /* logits and dlogits: AVEY_F32, AVEY_F16 or AVEY_BF16 */
  int32_t score;        /* AVEY_SCORE_* */
  int32_t renormalize;
  int32_t k;            /* 1..32 */
  int32_t groups;       /* 1..32, a divisor of experts */
  int32_t top_groups;   /* 1..groups */
  int32_t group_best;   /* 1 or 2 */
  int64_t tokens, experts; /* up to 2^30 and 1024 */
  double scale;
  const void* logits;
  int64_t logits_ld;
  const float* bias;    /* [experts], or NULL */
  float* weights;       /* [tokens][k] (backward: as the forward call wrote it) */
  int32_t* chosen;      /* [tokens][k] (the same) */
  const float* dweights; /* backward: [tokens][k] */
  void* dlogits;         /* backward: contiguous [tokens][experts] */
} AveyRouteParams;

AVEY_API int avey_route_fwd_v1(const AveyRouteParams* params, void* stream);
AVEY_API int avey_route_bwd_v1(const AveyRouteParams* params, void* stream);

/*
 * Places of choices sorted by expert: slots[i] is the place of entry i among all entries
 * in the order of their experts (entries of one expert in their given order), and
 * expert e's entries hold the places [offsets[e], offsets[e + 1]). Entries with a number
 * outside [0, experts) hold the places from offsets[experts] on: they belong to no
 * expert (avey_linear_* gives zeros there).
 */
typedef struct AveyArrangeParams {
  uint32_t struct_size; /* sizeof(AveyArrangeParams) */
  int32_t index_bits;   /* 32 or 64: signed expert numbers */
  int64_t count, experts; /* up to 2^30 and 1024 */
  const void* chosen;   /* [count] */
  int32_t* slots;       /* [count] */
  int32_t* offsets;     /* [experts + 1] */
  void* workspace;      /* 256-byte aligned, >= avey_arrange_workspace_size() bytes */
  uint64_t workspace_bytes;
} AveyArrangeParams;

AVEY_API int avey_arrange_v1(const AveyArrangeParams* params, void* stream);
AVEY_API int avey_arrange_workspace_size(const AveyArrangeParams* params, uint64_t* bytes);

/*
 * Rows of tokens to the places of their choices and back, with slots [tokens][k] that
 * hold each place in [0, tokens k) at most once (a slot outside it stands for no place: its
 * choice is left out; a place that no slot names gets zeros with `clear`, and is not written
 * without):
 *
 *   dispatch      rows[slots[t][j]] = x[t]
 *   combine       out[t] = x[t] (the residual, or 0 where x is NULL)
 *                          + sum_j weights[t][j] rows[slots[t][j]]  (weights NULL: 1)
 *   combine_bwd   drows[slots[t][j]] = weights[t][j] x[t], dweights[t][j] =
 *                 <x[t], rows[slots[t][j]]>, with x the gradient of out
 *
 * dispatch's gradient is combine without weights and residual. Sums are fp32, in the
 * order of j, and rounded once.
 */
typedef struct AveyRowsParams {
  uint32_t struct_size; /* sizeof(AveyRowsParams) */
  int32_t dtype;        /* x, rows, out, drows: AVEY_F32, AVEY_F16 or AVEY_BF16 */
  int32_t k;            /* 1..32 */
  int32_t clear;        /* dispatch, combine_bwd: zeros for the places that no slot names */
  int64_t tokens, width; /* tokens x k up to 2^30, width up to 2^22 */
  const int32_t* slots;
  const void* x;
  int64_t x_ld;
  void* rows;           /* dispatch writes them */
  int64_t rows_ld;
  const float* weights; /* contiguous [tokens][k] */
  void* out;            /* combine: contiguous [tokens][width] */
  void* drows;          /* combine_bwd: contiguous [tokens k][width], or NULL */
  float* dweights;      /* combine_bwd: contiguous [tokens][k], or NULL */
  void* workspace;      /* with clear: 256-byte aligned, >= avey_rows_workspace_size() bytes */
  uint64_t workspace_bytes;
} AveyRowsParams;

/* Bytes of `workspace`: 0 without `clear` and up to 8192 places, else 4 a place. (A block that ends
 * before `workspace` is taken too, as one without `clear`.) */
AVEY_API int avey_rows_workspace_size(const AveyRowsParams* params, uint64_t* bytes);

AVEY_API int avey_dispatch_v1(const AveyRowsParams* params, void* stream);
AVEY_API int avey_combine_v1(const AveyRowsParams* params, void* stream);
AVEY_API int avey_combine_bwd_v1(const AveyRowsParams* params, void* stream);

/*
 * Embedding: out[i] = scale table[tokens[i]], rounded once (a token outside [0, vocab)
 * gives a row of NaN), and the table's gradient
 *
 *   dtable[v] = scale * (sum of dy[i] over the i with tokens[i] = v, in fp32)
 *
 * for every v, with zeros for tokens that do not occur, for `padding` (when it is not
 * negative) and for tokens outside the vocabulary. The tokens are sorted and each
 * sum is taken in one order: results are bitwise reproducible.
 */
typedef struct AveyEmbeddingParams {
  uint32_t struct_size; /* sizeof(AveyEmbeddingParams) */
  int32_t dtype;        /* table, out, dy, dtable: AVEY_F32, AVEY_F16 or AVEY_BF16 */
  int32_t index_bits;   /* 32 or 64: signed tokens */
  int32_t reserved;
  int64_t count, width, vocab; /* up to 2^30, 2^22 and 2^30 */
  int64_t padding;      /* a token without a gradient, or negative */
  double scale;
  const void* tokens;   /* [count] */
  const void* table;    /* forward */
  int64_t table_ld;
  void* out;            /* forward: contiguous [count][width] */
  const void* dy;       /* backward */
  int64_t dy_ld;
  void* dtable;         /* backward: contiguous [vocab][width] */
  void* workspace;      /* backward: 256-byte aligned, >= avey_embedding_workspace_size() bytes */
  uint64_t workspace_bytes;
} AveyEmbeddingParams;

AVEY_API int avey_embedding_fwd_v1(const AveyEmbeddingParams* params, void* stream);
AVEY_API int avey_embedding_bwd_v1(const AveyEmbeddingParams* params, void* stream);

/* Bytes of the backward call's `workspace`, at most: 32 a token for the sort, and for the parts of
 * runs of one token a byte for every element of dy (its tokens filled up to 8), or for every 4 from 18944
 * tokens on (up to 32); 4 KB. */
AVEY_API int avey_embedding_workspace_size(const AveyEmbeddingParams* params, uint64_t* bytes);

/*
 * One AdamW step over many tensors (no counterpart in the reference, which
 * leaves training to torch). For every element of every tensor, in fp32:
 *
 *   g = grad * (*grad_scale, or 1)
 *   m = beta1 m + (1 - beta1) g
 *   v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay)
 *         - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 *
 * p is master where given (param is then its rounding to dtype), else param.
 *
 * state_bits 32: exp_avg and exp_avg_sq are floats (m and v).
 *
 * state_bits 8: exp_avg and exp_avg_sq are float8 e4m3 codes of m and of
 * sqrt(v), in blocks of 256 consecutive elements (the last one of a tensor may
 * be shorter) with one float per block in exp_avg_scale / exp_avg_sq_scale:
 * value = code * scale, scale = max |value| / 448 (at least 2^-126). A new
 * value x is rounded stochastically: r = |x| (1 / scale), to which 20 random
 * bits are added below the last kept bit (r + 2^-6 in place of r below 2^-6,
 * where e4m3 is evenly spaced), and the rest is cut off. The bits of element i
 * of the call (tensors in order, each counted in whole blocks of 256) are
 *   h = mix(low32(i) ^ key), noise = 16 (h mod 2^16) + 8 for m and
 *   16 (h / 2^16) + 8 for sqrt(v),
 *   key = mix2(seed + 0x9e3779b9 (step + high32(i))) (all mod 2^32),
 * where mix is x ^= x >> 16; x *= 0x7feb352d; x ^= x >> 15; x *= 0x846ca68b;
 * x ^= x >> 16 and mix2 is x = (x ^ x >> 16) * 0x7feb352d, x = (x ^ x >> 16) *
 * 0x846ca68b (constants from C. Wellons, "Prospecting for hash functions", 2018).
 * The same call gives the same bits. A block that gets a
 * non-finite value has non-finite or undefined states from then on.
 */
#define AVEY_ADAMW_BLOCK 256

typedef struct AveyAdamWTensor {
  void* param;             /* dtype, numel elements */
  const void* grad;        /* dtype */
  void* exp_avg;           /* float, or e4m3 codes */
  void* exp_avg_sq;        /* float, or e4m3 codes of the square root */
  float* exp_avg_scale;    /* state_bits 8: ceil(numel / 256) floats */
  float* exp_avg_sq_scale; /* state_bits 8: ceil(numel / 256) floats */
  float* master;           /* numel floats, or NULL (for all tensors or none) */
  int64_t numel;           /* >= 0 */
} AveyAdamWTensor;

typedef struct AveyAdamWParams {
  uint32_t struct_size;   /* sizeof(AveyAdamWParams) */
  int32_t dtype;          /* AVEY_F32, AVEY_F16 or AVEY_BF16: param and grad */
  int32_t state_bits;     /* 32 or 8 */
  int32_t count;          /* tensors */
  const AveyAdamWTensor* tensors; /* host array */
  double lr, beta1, beta2, eps, weight_decay;
  int64_t step;           /* >= 1 */
  uint64_t seed;          /* state_bits 8 (low 32 bits are used) */
  const float* grad_scale; /* device float that multiplies every gradient, or NULL */
} AveyAdamWParams;

/* Enqueue the step on `stream`: one launch for every 400 tensors. The arrays
 * of a call must not overlap. */
AVEY_API int avey_adamw_v1(const AveyAdamWParams* params, void* stream);

/* Bytes of `workspace` the backward steps need for these parameters. */
AVEY_API int avey_bwd_workspace_size(const AveyBwdParams* params, uint64_t* bytes);

/* Message for the last non-OK status returned on this thread ("" if none). */
AVEY_API const char* avey_last_error(void);

/* Device-side status word of the current device: 0, or the OR of the
 * AVEY_DEVFLAG_* bits raised by kernels since the last clear. Synchronises
 * the device. clear != 0 resets it. */
#define AVEY_DEVFLAG_TIMEOUT 1u /* a bounded wait on an mbarrier gave up */
AVEY_API int avey_device_status(uint32_t* flags, int clear);

/* Number of kernels this library has launched in this process. */
AVEY_API uint64_t avey_launch_count(void);

/* Test-only hooks of the failure path (no counterpart in the reference).
 * wait_limit_cycles: SM cycles after which a bounded wait on an mbarrier gives
 * up (<= 0 restores the default of about one second). stall != 0: later
 * launches of the fused tensor-core kernel start with their TMA and MMA warps
 * issuing nothing, and those of the linear layers and the cross entropy with their TMA
 * lanes issuing nothing, so the first wait for their work runs out, the kernel
 * raises AVEY_DEVFLAG_TIMEOUT, unwinds and returns (no trap, the context stays
 * usable). The wait limit applies to the current device; the stall flag to
 * the process. Not for production use. */
AVEY_API int avey_test_hooks_v1(long long wait_limit_cycles, int stall);

/* AVEY_ABI_VERSION of the loaded library. */
AVEY_API int avey_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* AVEY_B200_H */
