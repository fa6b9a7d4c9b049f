/*
 * axhip.h -- C ABI of the gfx950 (MI355X) GPU backend for Axiom's two GPU hot
 * paths: scaled-dot-product attention and the fused elementwise / softmax /
 * norm chains that the lazy graph emits.
 *
 * Conventions
 *   - every function returns int: 0 on success, a positive value is a
 *     hipError_t, a negative value is one of AXHIP_ERR_*.  A human-readable
 *     message for the calling thread's last failure is at axhip_last_error().
 *   - the caller owns every buffer; kernels never allocate.  Pointers are
 *     device pointers unless a parameter says "host".  Six entry points need
 *     temporary device memory for some argument values (axhip_sdpa_fwd,
 *     axhip_sdpa_packed, axhip_sdpa_paged, axhip_gemm, axhip_argreduce,
 *     axhip_reduce_axis: each says when).  Their
 *     *_ws forms take it from the caller -- `workspace` of at least
 *     *_workspace_bytes(...) bytes, 256-byte aligned -- and allocate nothing;
 *     the plain forms (and a *_ws call with workspace == NULL) take it from the
 *     stream-ordered allocator (hipMallocAsync / hipFreeAsync on `stream`), a
 *     convenience that graph capture and no-allocation harnesses must avoid.
 *     A workspace that is too small fails with AXHIP_ERR_WORKSPACE before
 *     anything is launched.
 *   - `stream` is a hipStream_t passed as void* (NULL = the backend's own
 *     stream, created by axhip_init and shared process-wide).
 *   - no exception crosses this boundary.
 *
 * Each entry point names the Axiom interface it stands behind (paths relative
 * to the Axiom source tree).
 */
#ifndef AXHIP_H
#define AXHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AXHIP_OK 0
#define AXHIP_ERR_INVALID_ARG (-1)
#define AXHIP_ERR_UNSUPPORTED (-2)
#define AXHIP_ERR_NO_DEVICE (-3)
#define AXHIP_ERR_WORKSPACE (-4)

/* element types (DType subset of include/axiom/dtype.hpp:171-191) */
#define AXHIP_DTYPE_F32 0
#define AXHIP_DTYPE_F16 1
#define AXHIP_DTYPE_BF16 2
/* Bool / UInt8 (one byte; any nonzero byte reads as 1.0, a nonzero result is stored as 1): the result type of
 * comparisons, logical operations and any / all, and an input type of the fused chains and of axhip_strided_copy
 * and axhip_where.  Attention, GEMM and the other entry points take the three floating-point types only. */
#define AXHIP_DTYPE_U8 3

/* ------------------------------------------------------------------ runtime
 * Stands behind system::is_metal_available (src/tensor/system.cpp:11-29),
 * make_storage(bytes, Device::GPU) (src/tensor/storage.cpp:26-48),
 * MetalStorage::copy_to/copy_from (src/backends/metal/metal_storage.mm:66-142)
 * and MetalExecutionStream::synchronize (src/backends/metal/metal_common.mm:
 * 285-335).  The Apple unified-memory retag (src/tensor/tensor.cpp:1600-1623)
 * has no counterpart: transfers are explicit hipMemcpyAsync. */
int axhip_device_count(int *count);
int axhip_init(int device);
const char *axhip_last_error(void);
const char *axhip_version(void);
void *axhip_default_stream(void);
int axhip_malloc(void **ptr, size_t bytes);
int axhip_free(void *ptr);
int axhip_memcpy_h2d_async(void *dst_device, const void *src_host, size_t bytes, void *stream);
int axhip_memcpy_d2h_async(void *dst_host, const void *src_device, size_t bytes, void *stream);
int axhip_memcpy_d2d_async(void *dst_device, const void *src_device, size_t bytes, void *stream);
int axhip_stream_sync(void *stream);

/* --------------------------------------------------------------------- SDPA
 * Stands behind backends::metal::gpu_scaled_dot_product_attention
 * (src/backends/metal/metal_operations.hpp:47-50, dispatch in
 * src/backends/metal/flash_attention_dispatch.mm:168-304, kernel
 * src/backends/metal/flash_attention.metal:50-224), called from
 * ops::scaled_dot_product_attention (src/tensor/operations.cpp:3979-4044).
 *
 * q (B,H,Sq,D), k/v (B,H,Skv,D), o (B,H,Sq,D).  The last dimension is
 * contiguous; the other three carry explicit element strides so the
 * (B,S,H,D)->(B,H,S,D) head-split view of nn::MultiHeadAttention
 * (src/nn/attention.cpp:44-52) needs no copy.  mask is NULL or uint8,
 * nonzero = masked out (include/axiom/operations.hpp:650), laid out
 * (Sq,Skv) row-major per (batch, head) with element strides mask_strides
 * (0 = broadcast).  is_causal masks kv_pos > q_pos (top-left aligned,
 * src/backends/cpu/flash_attention_cpu.cpp:78-89).  scale <= 0 means
 * 1/sqrt(D) (src/tensor/operations.cpp:4013-4015).  A row whose keys are all
 * masked yields zeros.  K may hold anything, infinities and NaN too, where a
 * key is masked; V there meets a weight of zero and has to be finite (a block
 * of keys that no row of a tile sees may not be read at all).  fp32
 * accumulation; output in `dtype`.
 * bf16/f16 with D a multiple of 8 up to 256, and fp32 with D a multiple of
 * 4 up to 128, run on MFMA (16-byte aligned base
 * pointers, strides that are multiples of 8 elements; fp32: 4); everything
 * else up to D = 256 runs on the generic fp32-FMA kernel, which takes the
 * place of the reference's decomposed_attention fallback
 * (flash_attention_dispatch.mm:125-162).  axhip_sdpa_kernel_name tells which.
 * A decoding step (up to 128 query rows, at most 96 (batch, head) slices, a
 * long unmasked key sequence) splits its keys between work-groups and merges
 * the partial results through stream-ordered temporary memory
 * (hipMallocAsync on `stream`). */
typedef struct {
    int32_t dtype;
    int32_t batch, heads, seq_q, seq_kv, head_dim;
    float scale;
    int32_t is_causal;
    int64_t q_strides[3]; /* batch, head, seq (elements) */
    int64_t k_strides[3];
    int64_t v_strides[3];
    int64_t o_strides[3];
    int64_t mask_strides[2]; /* batch, head (elements; 0 = shared) */
} AxhipSdpaParams;

int axhip_sdpa_fwd(const void *q, const void *k, const void *v, void *o,
                   const uint8_t *mask, const AxhipSdpaParams *params_host, void *stream);
/* The same with the temporary memory of a decoding step handed in by the
 * caller (the role of the reference's caller-owned command buffers,
 * src/backends/metal/metal_common.hpp:53-123: the backend allocates nothing
 * behind the caller's back).  axhip_sdpa_workspace_bytes answers 0 for every
 * problem that needs none; has_mask: whether a mask will be passed.  Steps of
 * fewer than 8 M key elements (slices x keys x dims) only run faster with it:
 * without one, or with less, they run undivided and allocate nothing.  So do
 * 16-bit problems of 24 M scores and more under a mask whose packing to bits
 * pays (one that (batch, head) slices share; one per slice of few or very many
 * rows), which take it for the mask as bits. */
size_t axhip_sdpa_workspace_bytes(const AxhipSdpaParams *params_host, int has_mask);
int axhip_sdpa_fwd_ws(const void *q, const void *k, const void *v, void *o,
                      const uint8_t *mask, const AxhipSdpaParams *params_host,
                      void *workspace, size_t workspace_bytes, void *stream);
/* name of the kernel axhip_sdpa_fwd would launch for these parameters
 * ("mfma_bf16_d128", "generic", ...); the pointer stays valid for the life of
 * the process. */
const char *axhip_sdpa_kernel_name(const AxhipSdpaParams *params_host);
/* diagnostic: the schedule the calling thread's last axhip_sdpa_fwd launched ("pingpong", "pipelined8",
 * "pipelined4", "key_split", "key_split8", "decode_split", "direct", "register_staged", "mfma_f32", "generic", "empty"; several
 * schedules share one kernel name; "mfma_f32_1", "_2" and "_4": fp32 with that many waves to 32 query rows where it
 * is not their number that says so).  AXHIP_SDPA_PINGPONG=0 in the environment (read when the library loads)
 * sends "pingpong" problems to "pipelined4" or "pipelined8". */
const char *axhip_sdpa_last_schedule(void);

/* ------------------------------------------------------------ fused chains
 * Stands behind graph::materialize_gpu_graph (called from
 * src/graph/graph_registry.cpp:834-850, Metal implementation
 * src/backends/metal/mpsgraph_graph_compiler.mm:706-944), the CPU-planned
 * hooks execute_gpu_fused_chain / execute_gpu_fused_reduction
 * (include/axiom/graph/gpu_fusion.hpp:14-22), the norm fast paths
 * gpu_layer_norm / gpu_rms_norm (src/backends/metal/metal_operations.hpp:
 * 20-24; kernels src/backends/metal/kernels.metal:167-381,
 * src/backends/metal/mpsgraph_operations.mm:2139-2210) and the per-op GPU
 * registry entries (src/backends/metal/mpsgraph_operations.mm:2925-3150).
 *
 * A program describes ONE pass over a [rows, cols] row-major view:
 *     v = input
 *     v = pre[0..n_pre)(v)            elementwise chain
 *     v = row_op(v)                   softmax / log-softmax / layer norm / RMS norm over cols
 *     v = post[0..n_post)(v)          elementwise chain
 *     out = reduce(v) over cols       -> [rows], or out = v -> [rows, cols]
 * Every value is computed in fp32 and rounded once on store.  One kernel
 * launch, each input element read once, no intermediate ever written.
 *
 * Chain op codes follow ops::OpType (include/axiom/operations.hpp:55-208) for
 * the hot-path subset. */
#define AXHIP_OP_ADD 1
#define AXHIP_OP_SUB 2
#define AXHIP_OP_MUL 3
#define AXHIP_OP_DIV 4
#define AXHIP_OP_MAX 5
#define AXHIP_OP_MIN 6
#define AXHIP_OP_RSUB 7 /* operand - v  (chain value is the right-hand side) */
#define AXHIP_OP_RDIV 8 /* operand / v */
#define AXHIP_OP_RELU 16
#define AXHIP_OP_GELU 17
#define AXHIP_OP_SQRT 18
#define AXHIP_OP_EXP 19
#define AXHIP_OP_NEG 20
#define AXHIP_OP_ABS 21
#define AXHIP_OP_SIGMOID 22
#define AXHIP_OP_TANH 23
#define AXHIP_OP_SILU 24
#define AXHIP_OP_LOG 25
#define AXHIP_OP_SQUARE 26
#define AXHIP_OP_RSQRT 27
#define AXHIP_OP_RECIP 28
/* The wider operator table of the lazy graph (binary: 40-63, unary: 64-95), with the CPU functors' rules
 * (src/backends/cpu/cpu_operations.hpp:214-235 power / fmod, :237-291 comparisons and logical operations, :360-381
 * atan2 / hypot, :395-400 logical not, :497-505 erf, :655-660 leaky ReLU, :724-787 sign / floor / ceil / trunc /
 * round, :808-860 cbrt / isnan / isinf / isfinite).  Comparisons, logical operations and the is* tests yield 1.0 or
 * 0.0 inside a chain; stored to an AXHIP_DTYPE_U8 output that is the reference's Bool result.  A logical operation
 * reads any nonzero value (NaN included) as true. */
#define AXHIP_OP_POW 40    /* powf(v, operand) */
#define AXHIP_OP_RPOW 41   /* powf(operand, v) */
#define AXHIP_OP_MOD 42    /* fmodf(v, operand): the sign of the dividend, like the CPU functor */
#define AXHIP_OP_RMOD 43   /* fmodf(operand, v) */
#define AXHIP_OP_ATAN2 44  /* atan2f(v, operand) */
#define AXHIP_OP_RATAN2 45 /* atan2f(operand, v) */
#define AXHIP_OP_HYPOT 46
#define AXHIP_OP_EQ 47
#define AXHIP_OP_NE 48
#define AXHIP_OP_LT 49 /* v < operand; with the chain value on the right-hand side the planner emits GT */
#define AXHIP_OP_LE 50
#define AXHIP_OP_GT 51
#define AXHIP_OP_GE 52
#define AXHIP_OP_AND 53
#define AXHIP_OP_OR 54
#define AXHIP_OP_XOR 55
#define AXHIP_OP_LEAKY_RELU 56 /* v > 0 ? v : operand * v -- the slope is the operand (an immediate) */
#define AXHIP_OP_ERF 64
#define AXHIP_OP_SIN 65
#define AXHIP_OP_COS 66
#define AXHIP_OP_TAN 67
#define AXHIP_OP_SIGN 68 /* 1, -1, or 0 (also for NaN) */
#define AXHIP_OP_FLOOR 69
#define AXHIP_OP_CEIL 70
#define AXHIP_OP_ROUND 71 /* halves away from zero (std::round) */
#define AXHIP_OP_TRUNC 72
#define AXHIP_OP_CBRT 73
#define AXHIP_OP_ISNAN 74
#define AXHIP_OP_ISINF 75
#define AXHIP_OP_ISFINITE 76
#define AXHIP_OP_NOT 77 /* v == 0 */

#define AXHIP_ROWOP_NONE 0
#define AXHIP_ROWOP_SOFTMAX 1
#define AXHIP_ROWOP_LOGSOFTMAX 2
#define AXHIP_ROWOP_LAYERNORM 3 /* (x-mean)/sqrt(var+eps) [*w] [+b], population variance */
#define AXHIP_ROWOP_RMSNORM 4   /* x/sqrt(mean(x^2)+eps) [*w] */

#define AXHIP_RED_NONE 0
#define AXHIP_RED_SUM 1
#define AXHIP_RED_MEAN 2
#define AXHIP_RED_MAX 3
#define AXHIP_RED_MIN 4
#define AXHIP_RED_PROD 5 /* (any / all are NE 0 under MAX / MIN with an AXHIP_DTYPE_U8 result) */

/* how a binary op's second operand maps onto the [rows, cols] view */
#define AXHIP_BK_FULL 0   /* [rows, cols] */
#define AXHIP_BK_ROWVEC 1 /* [cols]  broadcast down the rows (weights, biases) */
#define AXHIP_BK_COLVEC 2 /* [rows]  one value per row (keep_dims reductions) */
#define AXHIP_BK_SCALAR 3 /* [1]     Axiom's make_scalar operand, device resident */
#define AXHIP_BK_IMM 4    /* immediate in AxhipChainOp.imm, no memory operand */

#define AXHIP_MAX_CHAIN 16
#define AXHIP_MAX_OPERANDS 8

typedef struct {
    const void *ptr;
    int32_t dtype;
    int32_t kind; /* AXHIP_BK_* */
} AxhipOperand;

typedef struct {
    int32_t op;      /* AXHIP_OP_* */
    int32_t operand; /* index into operands[] for binary ops, -1 otherwise */
    float imm;       /* value for AXHIP_BK_IMM */
    int32_t imm_kind; /* AXHIP_BK_IMM when imm is the operand, else 0 */
} AxhipChainOp;

typedef struct {
    int64_t rows, cols;
    const void *input;
    int32_t input_dtype;
    int32_t n_operands;
    AxhipOperand operands[AXHIP_MAX_OPERANDS];
    int32_t n_pre;
    AxhipChainOp pre[AXHIP_MAX_CHAIN];
    int32_t row_op; /* AXHIP_ROWOP_* */
    float eps;
    int32_t norm_weight; /* operand index (ROWVEC) or -1 */
    int32_t norm_bias;   /* operand index (ROWVEC) or -1 */
    int32_t n_post;
    AxhipChainOp post[AXHIP_MAX_CHAIN];
    int32_t reduce; /* AXHIP_RED_* over cols */
    void *output;   /* [rows] if reduce != NONE else [rows, cols] */
    int32_t output_dtype;
} AxhipRowsProgram;

int axhip_fused_rows(const AxhipRowsProgram *program_host, void *stream);
/* name of the kernel variant axhip_fused_rows would launch: "rows_static_..." a kernel of
 * this program shape built into the library, "rows_jit_..." one the library compiles (hipRTC)
 * when the shape is first launched -- the counterpart of the reference compiling a graph on
 * first use (mpsgraph_graph_compiler.mm:706-944) -- anything else the generic interpreter.
 * AXHIP_JIT=0 in the environment turns run-time compilation off. */
const char *axhip_fused_rows_kernel_name(const AxhipRowsProgram *program_host);
/* Compiles the kernel of a "rows_jit_" program now (for gfx950; needs no device) and reports
 * a compile error instead of leaving it to the first launch, which would fall back to the
 * interpreter.  Pointers in the program are only looked at for their alignment. */
int axhip_fused_rows_prepare(const AxhipRowsProgram *program_host);
/* diagnostic: how many "rows_jit_" kernels this process has so far loaded from the on-disk cache of
 * compiled code objects (AXHIP_CACHE_DIR, default $XDG_CACHE_HOME/axhip or $HOME/.cache/axhip; AXHIP_DISK_CACHE=0
 * turns it off) and how many it compiled with hipRTC.  Either pointer may be NULL. */
void axhip_fused_rows_jit_counters(int *from_disk, int *compiled);

/* Elementwise chain followed by a reduction over ALL elements -> one value
 * (the FusedReductionStep of include/axiom/graph/compiled_graph.hpp:41-70,
 * GPU hook execute_gpu_fused_reduction).  Uses program->pre only; row_op and
 * post must be empty; program->reduce selects the reduction; output is one
 * element.  workspace: device scratch of at least
 * axhip_full_reduce_workspace_bytes() bytes. */
size_t axhip_full_reduce_workspace_bytes(void);
int axhip_fused_full_reduce(const AxhipRowsProgram *program_host, void *workspace,
                            size_t workspace_bytes, void *stream);

/* axhip_fused_full_reduce for callers that cannot allocate device memory or
 * bring a workspace: code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc.  It has no counterpart in the reference.
 * Same program, same kernels and the same result, bit for bit; the partial
 * sums live in a 65 KiB array inside the library's device image (one copy on
 * every device the library runs on, held until the process ends), whose
 * address is resolved when axhip_init runs on the device.  The call itself
 * performs no hipMalloc / hipFree, calls no allocating routine and compiles
 * nothing (only kernels that are built into the library serve it).
 * Limits: rows * cols <= axhip_full_reduce_noalloc_max_elements() (2^40),
 * larger inputs return AXHIP_ERR_UNSUPPORTED.  All calls on one device share
 * that one array: two calls that overlap in time on the same device (different
 * streams, or different threads on different streams) race; calls on one
 * stream are ordered and safe.  Nothing in the array has to be cleared
 * between calls. */
int64_t axhip_full_reduce_noalloc_max_elements(void);
int axhip_fused_full_reduce_noalloc(const AxhipRowsProgram *program_host, void *stream);

/* ------------------------------------------------------------- data movers
 * Stands behind gpu_make_contiguous (src/backends/metal/metal_operations.hpp:
 * 60-63, kernel gather_strided src/backends/metal/kernels.metal:33-149) and
 * the GPU Cast op (src/tensor/tensor.cpp:1665-1670).  Copies a strided view
 * (<= 8 dims, non-negative element strides) into a contiguous row-major
 * buffer, converting dtype on the way (AXHIP_DTYPE_U8 on either side: the
 * Bool casts, nonzero <-> 1). */
#define AXHIP_MAX_DIMS 8
int axhip_strided_copy(const void *src, int32_t src_dtype, void *dst, int32_t dst_dtype,
                       int32_t ndim, const int64_t *shape_host, const int64_t *src_strides_host,
                       void *stream);
int axhip_fill(void *dst, int32_t dtype, double value, int64_t count, void *stream);

/* Constant padding (ops::pad, mode "constant": src/tensor/operations.cpp pad();
 * lazy Pad node, src/backends/metal/mpsgraph_graph_compiler.mm:335-573).  dst is
 * contiguous row-major with extents src_shape[d] + pad_before[d] + pad_after[d];
 * src may be a strided view (non-negative element strides).  One pass: each
 * output element is either copied or set to `value`. */
int axhip_pad(const void *src, void *dst, int32_t dtype, int32_t ndim, const int64_t *src_shape_host,
              const int64_t *src_strides_host, const int64_t *pad_before_host,
              const int64_t *pad_after_host, double value, void *stream);
/* The other modes of ops::pad (src/tensor/operations.cpp:2216-2246): reflect
 * (the border element is not repeated; each pad must be shorter than the
 * extent it reflects), replicate (the border element repeated) and circular
 * (wrap around); `value` only matters for AXHIP_PAD_CONSTANT. */
#define AXHIP_PAD_CONSTANT 0
#define AXHIP_PAD_REFLECT 1
#define AXHIP_PAD_REPLICATE 2
#define AXHIP_PAD_CIRCULAR 3
int axhip_pad_mode(const void *src, void *dst, int32_t dtype, int32_t ndim, const int64_t *src_shape_host,
                   const int64_t *src_strides_host, const int64_t *pad_before_host,
                   const int64_t *pad_after_host, int32_t mode, double value, void *stream);

/* masked_fill (include/axiom/operations.hpp:437-440): dst[i] = mask[i] ? value :
 * src[i] over an iteration space of <= 8 dims; src and the byte mask (Bool:
 * nonzero = fill) are strided views with element strides, 0 on broadcast dims;
 * dst is contiguous and has src's dtype. */
int axhip_masked_fill(const void *src, int32_t dtype, const uint8_t *mask, void *dst, int32_t ndim,
                      const int64_t *shape_host, const int64_t *src_strides_host,
                      const int64_t *mask_strides_host, double value, void *stream);

/* where (ops::where, include/axiom/operations.hpp:425-429 and
 * src/tensor/operations.cpp:1543-1566; GPU MPSGraphTernaryOperation::execute_where,
 * src/backends/metal/mpsgraph_operations.mm:637): dst[i] = cond[i] != 0 ?
 * a[i] : b[i] over an iteration space of <= 8 dims.  cond (normally
 * AXHIP_DTYPE_U8), a and b are strided views with element strides, 0 on
 * broadcast dims, each of its own element type; dst is contiguous. */
int axhip_where(const void *cond, int32_t cond_dtype, const void *a, int32_t a_dtype, const void *b,
                int32_t b_dtype, void *dst, int32_t dst_dtype, int32_t ndim, const int64_t *shape_host,
                const int64_t *cond_strides_host, const int64_t *a_strides_host,
                const int64_t *b_strides_host, void *stream);

/* Embedding lookup (ops::embedding, include/axiom/operations.hpp:483-486):
 * dst[i, :] = table[indices[i], :] for n_indices rows of row_elems elements.
 * index_bytes is 4 (int32) or 8 (int64).  An index outside [0, table_rows)
 * yields a row of zeros (the device cannot throw IndexError). */
int axhip_gather_rows(const void *table, int32_t dtype, int64_t table_rows, int64_t row_elems,
                      const void *indices, int32_t index_bytes, int64_t n_indices, void *dst,
                      void *stream);

/* argmax (want_min = 0) / argmin along the middle extent of a contiguous
 * (outer, axis, inner) view -> outer * inner int64 indices: the Reduction node
 * kinds ArgMax / ArgMin of the GPU graph compiler
 * (src/backends/metal/mpsgraph_graph_compiler.mm:628-658), with the CPU scan's
 * rule (src/backends/cpu/cpu_operations.cpp:2157-2229): the first occurrence of
 * the extreme wins, a NaN never does, and a slice with nothing above the type's
 * lowest() (argmin: below max()) -- all -inf, all NaN -- answers 0.  inner == 1
 * is the row form (greedy decoding over [batch, vocabulary] logits).  Few
 * results over a long inner-axis run go through stream-ordered temporary
 * memory (hipMallocAsync on `stream`). */
int axhip_argreduce(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner,
                    int32_t want_min, int64_t *dst, void *stream);
/* The same with that temporary memory handed in by the caller (0 bytes for
 * every shape that needs none; `src` only matters for its 16-byte alignment). */
size_t axhip_argreduce_workspace_bytes(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner);
int axhip_argreduce_ws(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner,
                       int32_t want_min, int64_t *dst, void *workspace, size_t workspace_bytes, void *stream);

/* Sum / mean / max / min (AXHIP_RED_*) along the middle extent of a contiguous
 * (outer, axis, inner) view -> outer * inner values of dst_dtype: Reduction
 * nodes over axes other than the last one
 * (src/backends/metal/mpsgraph_graph_compiler.mm:576-604 reduces over any axes),
 * without a transposing copy.  fp32 accumulation; the mean divides by the axis
 * length.  inner == 1 is a row reduction and goes to the fused row kernels.
 * Few results over a long axis are reduced in two passes through fp32
 * partials in stream-ordered temporary memory (hipMallocAsync on `stream`). */
int axhip_reduce_axis(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner,
                      int32_t reduce, void *dst, int32_t dst_dtype, void *stream);
/* The same with the fp32 partials in memory handed in by the caller (0 bytes
 * for every shape that needs none; `src` only matters for its alignment). */
size_t axhip_reduce_axis_workspace_bytes(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner);
int axhip_reduce_axis_ws(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner,
                         int32_t reduce, void *dst, int32_t dst_dtype, void *workspace, size_t workspace_bytes, void *stream);

/* softmax (is_log = 0) / log-softmax along the middle extent of a contiguous
 * (outer, axis, inner) view, dst of the same shape and dtype (src itself, or
 * memory that does not overlap it): Softmax /
 * LogSoftmax nodes over an axis other than the last one
 * (src/backends/metal/mpsgraph_graph_compiler.mm:287-300 takes any axis),
 * without the two transposing copies.  inner == 1 goes to the fused row
 * kernels. */
int axhip_softmax_axis(const void *src, int32_t dtype, int64_t outer, int64_t axis, int64_t inner,
                       int32_t is_log, void *dst, void *stream);

/* -------------------------------------------------------------------- GEMM
 * Stands behind the GPU MatMul registry entry and gpu_linear
 * (src/backends/metal/mpsgraph_operations.mm:2409-2532; lazy builder
 * src/backends/metal/mpsgraph_graph_compiler.mm:271-284), used by nn::Linear
 * as matmul(x, W, false, true) + bias (src/nn/linear.cpp:15-27).
 * C[b] = op(A[b]) * op(B[b]) (+ bias[N]) (+ residual[b]) for b < batch;
 * row-major, lda/ldb/ldc and batch strides in elements (stride 0 shares an
 * operand across the batch).  fp32 accumulation; bf16/f16 on MFMA.
 * The matrix-core kernels read A along k (trans_a = 0) and B either way, at
 * any alignment.  A large product with A stored [k, m], and a large fp32 one
 * off the vector grid (k, or n of a B stored [k, n], not a multiple of 4)
 * where copying first is the faster way, is repacked: transposed, k
 * zero-padded, into temporary memory that the library takes and returns in
 * stream order (hipMallocAsync / hipFreeAsync on `stream`). */
typedef struct {
    int32_t dtype;
    int32_t trans_a, trans_b;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;
    int64_t batch;
    int64_t stride_a, stride_b, stride_c;
    const void *bias;     /* [n] or NULL */
    const void *residual; /* same layout as C or NULL */
    int32_t epilogue_op;  /* 0 or AXHIP_OP_RELU / GELU / SILU / SIGMOID / TANH (MatMul+activation fusion) */
} AxhipGemmParams;

int axhip_gemm(const void *a, const void *b, void *c, const AxhipGemmParams *params_host, void *stream);
/* The same with temporary memory handed in by the caller.  0 bytes below
 * 2^30 floating-point operations and for x W^T in whole 16-byte vectors; for
 * a large product with an operand stored the other way, or a k off that grid,
 * the size of the operands repacked -- also where the kernel that the product
 * gets reads them as they lie and leaves the memory alone.  Less is refused
 * with AXHIP_ERR_WORKSPACE; NULL leaves the allocation, if one is needed, to
 * the library. */
size_t axhip_gemm_workspace_bytes(const AxhipGemmParams *params_host);
int axhip_gemm_ws(const void *a, const void *b, void *c, const AxhipGemmParams *params_host,
                  void *workspace, size_t workspace_bytes, void *stream);
/* diagnostic: the kernel that the calling thread's last axhip_gemm or axhip_gemm_ws multiplied with: "skinny" (at most
 * eight rows), "big", "tile", "small" (16 bits), "f32_16x16" .. "f32_64x64", "ring_64x64", "ring_64x128" (fp32, by work-group
 * tile), the same with "_parts" (fp32 by products of bf16 parts), "fma", "empty". */
const char *axhip_gemm_last_kernel(void);

/* ------------------------------------------------------------- 8-bit rows
 * Rows of values as int8 with one fp32 scale each: q[r][j] * scales[r] stands for the value.  q lies in [-127, 127]; the nearest
 * integer is taken, halves to the even one, decided on exact products (a value next to a half falls on the right side of it; only of
 * a BFloat16 norm's row whose largest product lies below 2^-118 the products are those that fp32's subnormal numbers hold).
 * A row of zeros has scale 0; a row that holds an infinity or a NaN (or whose products overflow fp32) has scale NaN and zeros, so
 * that every product with it comes out as NaN.  Rows are contiguous, ld_* elements apart (at least cols; any alignment).
 *
 * axhip_quantize_q8: scales[r] = max_j |x[r][j]| / 127.  The weight (n, k) of nn::Linear by output channel, activations by token.
 *
 * axhip_rms_norm_q8: the residual's addition and the RMS norm of a pre-norm block (ops::add, then ops::rms_norm,
 * include/axiom/operations.hpp and src/nn/normalization.cpp), out in 8 bits for the product that follows: with
 *     h = x + residual, rounded to dtype (residual NULL: h = x),   y = h / sqrt(mean(h^2) + eps) * weight
 * q and scales stand for y, which is rounded nowhere else; the squares are summed up in 64 bits (of Float16 rows in 32), so that
 * rows whose squares are beyond fp32 have their scale too.  sum: NULL, or where h goes for the next residual addition (x or residual
 * itself, with the same ld, is allowed; needs a residual).  x, residual, weight (NULL: ones) and sum are of `dtype`.  No temporary
 * memory; axhip_quantize_q8 reads dtype, rows, cols, ld_x and ld_q only. */
typedef struct {
    int32_t dtype; /* of x, residual, weight and sum */
    float eps;
    int64_t rows, cols;
    int64_t ld_x, ld_residual, ld_sum, ld_q; /* elements */
} AxhipRowsQ8Params;

int axhip_quantize_q8(const void *x, int8_t *q, float *scales, const AxhipRowsQ8Params *params_host, void *stream);
int axhip_rms_norm_q8(const void *x, const void *residual, const void *weight, void *sum, int8_t *q, float *scales,
                      const AxhipRowsQ8Params *params_host, void *stream);

/* ------------------------------------------------------- products in 8 bits
 * nn::Linear (src/nn/linear.cpp:15-27) on rows in 8 bits: C = act(scale_a[m] scale_b[n] sum_k A[m][k] B[n][k] (+ bias[n]) (+ residual)),
 * A (m, k) and B (n, k) int8, row-major, lda / ldb / ldc in elements, any alignment.  The sums are int32 and exact: k up to
 * 131071, beyond which rows of -128 could overflow (AXHIP_ERR_UNSUPPORTED).  scale_a [m] and scale_b [n] are fp32; the rest is fp32 arithmetic (the sum as a
 * float times the scales' product, plus bias, rounded once; plus residual), the activation (of Float32 results within 2e-6 (1 + |y|) of its value y, of 16-bit ones within 2^-15 |y|, GELU
 * to BFloat16 within 2^-12 |y| and 2^-122), rounded once to dtype: a row of C has the same bits whatever the other rows are and however many (a NaN's own bits
 * aside).  What is not a number stays so under every activation.
 * residual has C's layout and may be C itself.  No temporary memory. */
typedef struct {
    int32_t dtype;       /* of C, bias and residual: Float32, Float16 or BFloat16 */
    int32_t epilogue_op; /* 0 or AXHIP_OP_RELU / GELU / SILU / SIGMOID / TANH */
    int64_t m, n, k;
    int64_t lda, ldb, ldc;
    const float *scale_a; /* [m] */
    const float *scale_b; /* [n] */
    const void *bias;     /* [n] or NULL */
    const void *residual; /* same layout as C or NULL */
} AxhipGemmQ8Params;

int axhip_gemm_q8(const int8_t *a, const int8_t *b, void *c, const AxhipGemmQ8Params *params_host, void *stream);
/* diagnostic: the kernel of the calling thread's last axhip_gemm_q8 */
const char *axhip_gemm_q8_last_kernel(void);

/* ---------------------------------------------------------------- sampling
 * A token from each row of logits [rows, vocab]: what axhip_argreduce does for greedy decoding, for the rest.  It has no
 * counterpart in the reference.  Each setting is an array of `rows` values on the device, or NULL (off); with `uniform` 1 the arrays are
 * NULL and the four values all_* hold for every row (nothing is allocated, copied or waited for on their behalf).  With
 * w_i = exp((l_i - max l) / temperature) and the order "larger logit first, equal ones by index":
 *     top_k  (k > 0)      keeps the first k;
 *     top_p  (p < 1)      of those, keeps the ones in front of which less than p of their sum of w lies (always the first);
 *     min_p  (0 < m)      of those, keeps the ones with w_i >= m (more than 1 counts as 1);
 *     u                   in [0, 1): the token is the first kept index, by index, at which the running sum of w exceeds u times
 *                         the sum of all that are kept.
 * temperature 0 (or less, or NaN) takes the first largest logit.  NULL: 1.  -inf and NaN are never drawn; +inf shares the draw with
 * its equals alone.  A row that has nothing else gets token -1.  probs (or NULL): the kept probability of the token (1 for
 * temperature 0, 0 for token -1).  The same arguments give the same tokens, whatever else runs: sums are of
 * multiples of 2^-43 of the largest weight, so that no order changes them; a token below 2^-44 of the most likely one is never drawn.
 * vocab up to 2^20 (AXHIP_ERR_UNSUPPORTED beyond), rows ld elements apart, any alignment. */
typedef struct {
    int32_t dtype;
    int32_t uniform; /* 0: the arrays; 1: the values at the end */
    int64_t rows, vocab, ld;
    const float *temperature; /* [rows] or NULL */
    const int32_t *top_k;     /* [rows] or NULL; 0 or less: off for the row */
    const float *top_p;       /* [rows] or NULL; 1 or more, or NaN: off for the row */
    const float *min_p;       /* [rows] or NULL; 0 or less, or NaN: off for the row */
    const float *u;           /* [rows] */
    float all_temperature;    /* read with uniform 1 only; off as in the arrays, temperature 1 being off */
    int32_t all_top_k;
    float all_top_p, all_min_p;
} AxhipSampleParams;

int axhip_sample(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params_host, void *stream);
/* The same with its temporary memory handed in by the caller.  Rows are drawn from in registers and LDS: 0 bytes for every shape, workspace may be NULL. */
size_t axhip_sample_workspace_bytes(const AxhipSampleParams *params_host);
int axhip_sample_ws(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params_host,
                    void *workspace, size_t workspace_bytes, void *stream);

/* -------------------------------------------- rotary positions and a cache
 * What a decoder does with positions and with the keys and values of its earlier tokens.  It has no counterpart in the reference,
 * whose attention takes keys that lie in one piece per (batch, head), of one length for the batch.
 *
 * Angles are fractions of a full turn in 64 bits: turns[i] = 2^64 f_i / (2 pi), f_i radians a position.  position * turns[i] modulo
 * 2^64 is then the angle of any position, a negative one too, to position * 2^-65 turns (2^-34 at position 2^31; a table of 32 bits is
 * position * 2^-33 off), and the kernels round it to 2^-33.
 * axhip_rope_turns fills such a table on the host (rot_dim / 2 values; no device is needed); copy it to the device once.  f_i =
 * theta^(-2 i / rot_dim), and for contexts longer than the trained `length`:
 *     LINEAR  f_i / factor
 *     BASE    theta * factor^(rot_dim / (rot_dim - 2)) in theta's place: the slowest angle is divided by factor, the fastest is kept
 *     BANDS   f_i (k + (1 - k) / factor), k = clamp((t - low) / (high - low), 0, 1), t = length f_i / (2 pi) the turns over `length`
 * theta >= 1; factor > 0; 0 <= low < high; length > 0.  What a kind does not name is not read. */
#define AXHIP_ROPE_PLAIN 0
#define AXHIP_ROPE_LINEAR 1
#define AXHIP_ROPE_BASE 2
#define AXHIP_ROPE_BANDS 3
typedef struct {
    int32_t rot_dim; /* even, up to 1024 */
    int32_t kind;    /* AXHIP_ROPE_* */
    double theta, factor, low, high, length;
} AxhipRopeScaling;
int axhip_rope_turns(const AxhipRopeScaling *scaling_host, uint64_t *turns_host);

/* y = x with the first rot_dim dims of every head rotated by its token's position, the other dims copied:
 *     y_a = amplitude (x_a cos t - x_b sin t),  y_b = amplitude (x_b cos t + x_a sin t)
 * over the pairs (a, b) = (i, i + rot_dim / 2), or (2 i, 2 i + 1) with `interleaved`.  `inverse` rotates back: with the same
 * amplitude it is the gradient of the call without it.  x, y: [tokens, heads, head_dim], the last dimension contiguous, element
 * strides of tokens and heads; y may be x itself (then with the same strides).  fp32 arithmetic (sines within 2^-22), rounded once. */
typedef struct {
    int32_t dtype;
    int32_t heads, head_dim, rot_dim; /* rot_dim: even, 2 .. head_dim */
    int32_t interleaved, inverse;     /* 0 or 1 */
    float amplitude;                  /* 0 means 1 */
    int32_t position_bytes;           /* 4 (int32) or 8 (int64) */
    int64_t tokens;
    int64_t x_strides[2], y_strides[2]; /* token, head (elements) */
    const void *positions;              /* [tokens] */
    const uint64_t *turns;              /* [rot_dim / 2], on the device */
} AxhipRopeParams;
int axhip_rope(const void *x, void *y, const AxhipRopeParams *params_host, void *stream);

/* The pages of a cache (of one layer): k and v are [n_pages, page_size rows, heads, head_dim] by element strides, in any order of
 * rows and heads, the last dimension contiguous.  Row j of a sequence lies in row j % page_size of page table[j / page_size], where
 * table is the sequence's row of a page table (int32, on the device).  page_size is a power of two up to 65536.  Offsets are 64 bits. */
typedef struct {
    void *k, *v;
    int32_t dtype;
    int32_t page_size;
    int32_t heads, head_dim;
    int64_t n_pages; /* below 2^31 */
    int64_t k_strides[3], v_strides[3]; /* page, row, head (elements) */
} AxhipKvPages;

/* New tokens into the cache, in one launch: q rotated to q_out as by axhip_rope (heads = 0: no q, q and q_out NULL; q_out may be q),
 * k rotated and v as it is written to row slots[t] % page_size of page slots[t] / page_size.  A slot that is negative or behind the
 * last page is not written (the padded end of a batch: q_out is written for it).  Two tokens must not have the same slot.  q, k, v,
 * q_out: [tokens, heads or pages.heads, head_dim] by token and head strides, such as views of one product's output.  rot_dim 0:
 * nothing is rotated, turns and positions may be NULL. */
typedef struct {
    AxhipKvPages pages;
    int32_t heads; /* of q: 0, or any number */
    int32_t rot_dim, interleaved;
    float amplitude;        /* of q and of k; 0 means 1 */
    int32_t position_bytes; /* 4 or 8 */
    int64_t tokens;
    int64_t q_strides[2], k_strides[2], v_strides[2], q_out_strides[2]; /* token, head (elements) */
    const void *positions;  /* [tokens] */
    const uint64_t *turns;  /* [rot_dim / 2], on the device */
    const int64_t *slots;   /* [tokens] */
} AxhipKvAppendParams;
int axhip_kv_append(const void *q, const void *k, const void *v, void *q_out, const AxhipKvAppendParams *params_host, void *stream);

/* Page dst[i] = page src[i], K and V of every layer: a fork's last page, a pool that is compacted.  With `rows`, the first rows[i]
 * rows only (values are clamped to 0 .. page_size).  A pair with a page that does not exist is left out; a page that one pair writes
 * may not be read or written by another one (a pair of a page and itself changes nothing). */
typedef struct {
    AxhipKvPages pages; /* of the first layer */
    int32_t layers;
    int32_t pairs;
    int64_t k_layer_stride, v_layer_stride; /* elements */
    const int32_t *src, *dst;               /* [pairs], on the device */
    const int32_t *rows;                    /* [pairs], on the device, or NULL: whole pages */
} AxhipKvCopyParams;
int axhip_kv_copy_pages(const AxhipKvCopyParams *params_host, void *stream);

/* Attention of packed sequences of different lengths.  q and o: [total_q, heads, head_dim] by token and head strides; sequence s owns
 * the rows cu_q[s] .. cu_q[s + 1] - 1 (rows of o that no sequence owns are left as they are).  Its keys are
 *   - the rows cu_kv[s] .. cu_kv[s + 1] - 1 of k and v, [total_kv, kv_heads, head_dim] by strides, or
 *   - with page_table (then k and v are NULL, cu_kv is not read): kv_lengths[s] rows of its pages, page_table[s * table_ld + ..].
 * heads is a multiple of kv_heads: head h reads key head h / (heads / kv_heads).  is_causal: the last query sees every key, the one in
 * front of it one less: query i of n sees key j <= i + keys - n, so that a sequence's next chunk of tokens can be computed behind what
 * the cache holds already.  A query that sees nothing yields zeros.  scale <= 0 means 1 / sqrt(head_dim).  fp32 sums and softmax, exponentials
 * rounded to dtype before the second product, results rounded once to dtype.
 * Keys outside a sequence are neither read nor can what lies there matter; a key that a causal query does not see meets a weight of zero and has to be finite in V.
 * Numbers in cu_q, cu_kv and kv_lengths that lie outside the tensors are clamped to them (total_q and total_kv below 2^30, keys of a
 * sequence up to 2^30); a page that does not exist makes NaN of every query that sees a key of it (of others of its sequence too, at times).
 * o may not overlap the inputs.  max_kv: about how many keys the longest sequence has, which the division of the work goes by and nothing else.  0 says that
 * they are few, not that nothing is known: one sequence of 8000 keys (a decoding step, 32 heads on 8 of 128) takes 83 us with it and 14 with 8000 or
 * more.  Where the host does not know lengths, give what there is room for (table_ld * page_size).
 * 16 bits with head_dim a multiple of 8 up to 256 and pages of 8 rows or more, 16-byte aligned, less than 4 GiB apart, on the matrix cores; fp32 with head_dim a multiple of 4 up to 128
 * likewise; everything else up to 256 dims on the generic kernel. */
typedef struct {
    int32_t dtype;
    int32_t heads, kv_heads, head_dim;
    int32_t n_seqs;
    int32_t is_causal;
    float scale;
    int32_t max_kv;
    int64_t total_q, total_kv;
    int64_t q_strides[2], k_strides[2], v_strides[2], o_strides[2]; /* token, head (elements) */
    const int32_t *cu_q;       /* [n_seqs + 1], on the device */
    const int32_t *cu_kv;      /* [n_seqs + 1] */
    const int32_t *page_table; /* [n_seqs, table_ld] or NULL */
    const int32_t *kv_lengths; /* [n_seqs] */
    int64_t table_ld;
    AxhipKvPages pages;        /* read with page_table only */
} AxhipSdpaPackedParams;
int axhip_sdpa_packed(const void *q, const void *k, const void *v, void *o, const AxhipSdpaPackedParams *params_host, void *stream);
size_t axhip_sdpa_packed_workspace_bytes(const AxhipSdpaPackedParams *params_host);
int axhip_sdpa_packed_ws(const void *q, const void *k, const void *v, void *o, const AxhipSdpaPackedParams *params_host,
                         void *workspace, size_t workspace_bytes, void *stream);

/* A decoding step: the last new_tokens tokens of each of n_seqs sequences against what the cache holds of it (theirs among it).  q and
 * o: [n_seqs, new_tokens, heads, head_dim] by strides; kv_lengths[s] keys in pages page_table[s * table_ld + ..]; token i sees key j <=
 * kv_lengths[s] - new_tokens + i.
 * Shared prefixes: the sequences group_starts[g] .. group_starts[g + 1] - 1 have the prefix_lengths[g] keys in pages
 * prefix_table[g * prefix_ld + ..] in front of their own, all of which every token sees.  They are read once for the group, not once
 * for each of its sequences.  Sequences in front of the first group and behind the last have no prefix; groups may be empty.
 * Everything else as in axhip_sdpa_packed; max_kv and max_prefix are hints alike (own keys, prefix), 0 among them.  Lengths, tables and groups are
 * read on the device when the kernels run: a captured step replays with what the arrays hold then. */
typedef struct {
    AxhipKvPages pages;
    int32_t heads;
    int32_t n_seqs, new_tokens;
    int32_t max_kv;
    float scale;
    int32_t n_groups; /* 0: no prefixes */
    int32_t max_prefix;
    int32_t reserved; /* 0 */
    int64_t q_strides[3], o_strides[3]; /* sequence, token, head (elements) */
    const int32_t *page_table;          /* [n_seqs, table_ld], on the device */
    const int32_t *kv_lengths;          /* [n_seqs] */
    int64_t table_ld;
    const int32_t *group_starts;        /* [n_groups + 1] */
    const int32_t *prefix_table;        /* [n_groups, prefix_ld] */
    const int32_t *prefix_lengths;      /* [n_groups] */
    int64_t prefix_ld;
} AxhipSdpaPagedParams;
int axhip_sdpa_paged(const void *q, void *o, const AxhipSdpaPagedParams *params_host, void *stream);
size_t axhip_sdpa_paged_workspace_bytes(const AxhipSdpaPagedParams *params_host);
int axhip_sdpa_paged_ws(const void *q, void *o, const AxhipSdpaPagedParams *params_host, void *workspace, size_t workspace_bytes,
                        void *stream);
/* diagnostic: the kernels of the calling thread's last axhip_sdpa_packed ("tile", "tile, eight waves", "tile, parts", "few", "few, parts";
 * fp32 "f32", "f32, apart", "f32, parts"; keys in parts are joined by a second launch) or axhip_sdpa_paged ("whole"; "shares", "shares, prefix":
 * joined alike); of either "generic" (head sizes and strides that the matrix-core kernels do not take), "empty". */
const char *axhip_sdpa_cache_last_kernel(void);

/* sizeof() of the parameter structs as this library was compiled, so that a
 * foreign-language binding can verify its own struct layout at load time:
 * which = 0 AxhipSdpaParams, 1 AxhipRowsProgram, 2 AxhipGemmParams,
 * 3 AxhipOperand, 4 AxhipChainOp, 5 AxhipRowsQ8Params, 6 AxhipGemmQ8Params,
 * 7 AxhipSampleParams, 8 AxhipRopeScaling, 9 AxhipRopeParams, 10 AxhipKvPages,
 * 11 AxhipKvAppendParams, 12 AxhipKvCopyParams, 13 AxhipSdpaPackedParams,
 * 14 AxhipSdpaPagedParams; anything else returns 0. */
size_t axhip_sizeof(int which);

#ifdef __cplusplus
}
#endif
#endif
