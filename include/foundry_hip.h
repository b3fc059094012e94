/*
 * foundry_hip.h: the C-ABI of libfoundry_hip.so, the MI355X (gfx950) backend
 * for Foundry's 4-bit quantized weight path.
 *
 * This is the one boundary a host binds. It is what the reference's `Device`
 * trait (src/nn/primitive.rs:70-120) needs from a backend, flattened to plain
 * pointers and sizes: a device owns one HIP stream; storage is device memory
 * the device allocated; every op returns a fresh output the caller allocated
 * and passes in. A Rust `src/hip` backend binds these through a thin FFI crate
 * (see INTEGRATION.md); the Python package foundry_amd binds them with ctypes.
 *
 * Conventions
 * - Every function returns an fh_status (0 = FH_OK). On error, fh_last_error()
 *   returns a thread-local message naming the function and the cause.
 * - Failure is sticky, as the reference's command stream is
 *   (src/metal/stream.rs:109-115, :201-212): once a launch or a
 *   synchronisation reports a device error, every later call on that device
 *   returns FH_ERR_FAILED.
 * - Ops validate shapes and dtypes before any launch (the reference does so in
 *   `primitive::output`, src/nn/primitive.rs:146-289) and check that every
 *   operand lies inside a live allocation of this device (the reference's
 *   ForeignStorage check, src/metal/mod.rs:187-200). A rejected call launches
 *   nothing.
 * - Ops are asynchronous on the device's stream. fh_download synchronises
 *   first (src/metal/mod.rs:614), fh_synchronize waits for everything.
 * - One host thread per device, as in the reference (Rc-based, !Send
 *   tensors). No internal locking.
 *
 * bf16 values are passed as their uint16_t bit patterns.
 */
#ifndef FOUNDRY_HIP_H
#define FOUNDRY_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FH_ABI_VERSION 2

typedef struct fh_device fh_device;
typedef struct fh_graph fh_graph;

/* Error kinds. Mirrors MetalError (src/metal/error.rs:7-58) where a HIP
 * counterpart exists, plus the Tensor-level validation errors
 * (src/nn/error.rs) that the reference raises before the device call. */
typedef enum fh_status {
    FH_OK = 0,
    FH_ERR_INVALID_ARGUMENT = 1,  /* shapes, sizes or null pointers do not fit the op */
    FH_ERR_DEVICE_UNAVAILABLE = 2,/* MetalError::DeviceUnavailable */
    FH_ERR_ALLOCATION = 3,        /* MetalError::BufferAllocation */
    FH_ERR_FOREIGN_STORAGE = 4,   /* MetalError::ForeignStorage */
    FH_ERR_OUT_OF_BOUNDS = 5,     /* MetalError::ToBytesOutOfBounds; operand past its allocation */
    FH_ERR_LAUNCH = 6,            /* a kernel launch was refused */
    FH_ERR_FAILED = 7,            /* MetalError::CommandBufferFailed (sticky) */
    FH_ERR_INDEX_TOO_LARGE = 8,   /* MetalError::KernelIndexTooLarge */
    FH_ERR_DTYPE = 9,             /* MetalError::DTypeNotFloat; TensorError::IndicesNotU32 */
    FH_ERR_UNSUPPORTED = 10,      /* valid request the kernels do not implement (e.g. group != 64) */
    FH_ERR_CAPTURE = 11           /* graph capture misuse */
} fh_status;

/* src/nn/dtype.rs:6-10 */
typedef enum fh_dtype { FH_F32 = 0, FH_BF16 = 1, FH_U32 = 2 } fh_dtype;

/* src/nn/profile.rs:7-13. STEPS keeps normal batching and times the span of
 * work; KERNELS brackets every dispatch with events (per-kernel GPU time). */
typedef enum fh_profile_mode {
    FH_PROFILE_OFF = 0,
    FH_PROFILE_STEPS = 1,
    FH_PROFILE_KERNELS = 2
} fh_profile_mode;

/* src/nn/memory.rs:1-5 */
typedef struct fh_allocated_memory {
    uint64_t bytes;
    const char *source; /* static string */
} fh_allocated_memory;

/* src/nn/profile.rs:15-21 (DeviceProfile) */
typedef struct fh_profile {
    uint64_t dispatches;      /* kernels launched since the last take */
    uint64_t allocations;     /* fh_alloc calls since the last take */
    uint64_t allocated_bytes; /* bytes they requested */
    uint64_t gpu_busy_ns;     /* union of timed GPU intervals (0 when unavailable) */
} fh_profile;

/* ---- errors and version ---- */
const char *fh_last_error(void);
int fh_abi_version(void);

/* ---- device lifecycle: MetalDevice::new / ::profiled (src/metal/mod.rs:108-149) ---- */
int fh_device_count(int *count);
int fh_device_create(int ordinal, fh_device **out);
int fh_device_create_profiled(int ordinal, int mode, fh_device **out);
/* Synchronises, frees every allocation the device still owns, destroys it. */
int fh_device_destroy(fh_device *dev);
/* Device::device_name (src/nn/primitive.rs:74) */
int fh_device_name(const fh_device *dev, char *buf, size_t len);
/* Device::synchronize (src/nn/primitive.rs:86) */
int fh_synchronize(fh_device *dev);
/* The device's HIP stream (hipStream_t), for callers that time with events. */
int fh_device_stream(fh_device *dev, void **stream);

/* ---- storage: Device::{zeros, storage_from_bytes, storage_to_bytes}
 *      (src/nn/primitive.rs:88-103; src/metal/mod.rs:565-637) ---- */
/* Allocates nbytes (at least 1) of device memory, 256-byte aligned. With
 * zero_fill != 0 the memory is cleared before any later op on the stream
 * reads it (Device::zeros). */
int fh_alloc(fh_device *dev, size_t nbytes, int zero_fill, void **out);
/* The same without the clearing, for storage that an op on the device's
 * stream writes before anything else touches it (an op's output): a block
 * kept for reuse is handed out without a wait for the work queued on it. */
int fh_alloc_output(fh_device *dev, size_t nbytes, void **out);
/* Frees an allocation of this device. The memory is given back to the driver,
 * or kept for later allocations of the device (at most 512 MiB, blocks of at
 * most 128 MiB, the oldest given back first, all of them when the driver runs
 * out), after the work queued on the GPU, on any stream, ends: the call itself
 * may return before.
 * A live graph retains every allocation its captured ops touched, as a
 * Metal command buffer retains its buffers (src/metal/mod.rs:280-282): the
 * allocation is then no longer usable by ops but stays allocated until the
 * last graph that uses it is destroyed. A free asked for while capturing is
 * carried out at fh_capture_end, on the same rule. */
int fh_free(fh_device *dev, void *ptr);
/* The same for memory that only ops on the device's stream (and fh_upload,
 * fh_download) have touched, such as an op's output that never left the
 * device: no other stream is waited for, since queued work that still uses it
 * runs before anything that a later owner enqueues. */
int fh_free_ordered(fh_device *dev, void *ptr);
/* Host -> device copy into an owned range; ordered on the stream. */
int fh_upload(fh_device *dev, void *dst, const void *src, size_t nbytes);
/* Device -> host copy of an owned range; synchronises first. */
int fh_download(fh_device *dev, void *dst, const void *src, size_t nbytes);

/* ---- memory and profile counters (src/nn/primitive.rs:75-83) ----
 * Bytes counted: every live allocation (including retired ones a graph still
 * holds) plus the device's own work areas (the 33 MB of GEMV/GEMM partial
 * sums and the batched GEMV's x image), allocated at creation; freed blocks
 * kept for reuse (fh_free, at most 512 MiB) are not counted. */
int fh_max_memory_allocated(const fh_device *dev, fh_allocated_memory *out);
int fh_reset_run_memory_peak(fh_device *dev);
int fh_run_memory_peak(const fh_device *dev, fh_allocated_memory *out);
/* Counters since the previous take, then reset. Returns FH_ERR_UNSUPPORTED
 * (and leaves *out zeroed) when the device was not created profiled, as the
 * reference returns None (src/nn/primitive.rs:83). */
int fh_take_profile(fh_device *dev, fh_profile *out);

/* ---- batching: the HIP counterpart of the reference's CommandStream
 * (src/metal/stream.rs:29-215), which encodes many dispatches and commits
 * them at once. Between begin and end, ops are validated and recorded, not
 * run; fh_graph_launch replays the recording on the device's stream. ---- */
int fh_capture_begin(fh_device *dev);
/* Ends the capture; the graph retains the allocations its ops touched. */
int fh_capture_end(fh_device *dev, fh_graph **out);
/* FH_ERR_FOREIGN_STORAGE for a graph of another (or a destroyed) device. */
int fh_graph_launch(fh_device *dev, fh_graph *graph);
/* Waits for the device's queued work (a replay may still be running), then
 * destroys the graph and releases its allocations; any the caller already
 * freed are freed now. A graph may outlive its device (it can then only be
 * destroyed). */
int fh_graph_destroy(fh_graph *graph);

/* ---- event timing on the device's stream ---- */
/* Records a start event now, in stream order. */
int fh_timer_begin(fh_device *dev);
/* Records an end event, waits for it, writes the milliseconds between the two. */
int fh_timer_end(fh_device *dev, double *elapsed_ms);

/* ---- the HBM read ceiling, for measurement: one launch that reads nbytes
 * (16-byte aligned, a multiple of 16) in 16-byte loads, 32 KB per block,
 * and writes one XOR word per wavefront to out (fh_read_probe_blocks gives
 * the number of words). No counterpart in the reference (it is the
 * roofline's measured read rate beside the quoted peak). ---- */
int fh_read_probe_blocks(uint64_t nbytes, uint64_t *blocks);
int fh_read_probe(fh_device *dev, const void *src, uint64_t nbytes, uint32_t *out);

/* ======================================================================
 * q4 ops. Weight format (affine group quantisation):
 *   wq     u32 [rows, k/8]   element j of a row = nibble j%8 (bits 4*(j%8)..+3)
 *                            of word j/8, little-endian nibble order
 *   scales bf16[rows, k/group]
 *   biases bf16[rows, k/group]
 *   w[r, j] = f32(scales[r, j/group]) * q[r, j] + f32(biases[r, j/group])
 * The kernels implement group = 64 and k a multiple of 64.
 * ====================================================================== */

/* q4 Embedding::forward (src/nn/linear.rs:53-69) -> Op::IndexSelect{dim 0}
 * (src/nn/primitive.rs:258-289; src/metal/mod.rs:483-500;
 * src/metal/kernels/index_select.metal:11-29) over a q4 table.
 * out bf16[n_ids, k]: out[i, :] = RNE_bf16(w[ids[i], :]); an id >= rows
 * writes a zero row. Bit-exact. n_ids may be 0. */
int fh_q4_embed(fh_device *dev, const uint32_t *wq, const uint16_t *scales,
                const uint16_t *biases, int64_t rows, int64_t k, int64_t group,
                const uint32_t *ids, int64_t n_ids, uint16_t *out);

/* q4 Linear::forward (src/nn/linear.rs:22-35) -> Op::Matmul
 * (src/nn/primitive.rs:234-256; src/metal/mod.rs:434-481;
 * src/metal/kernels/matmul.metal:29-65) with a q4 right operand:
 *   y[i, r] = sum_j x[i, j] * w[r, j]       (fp32 accumulation)
 * x bf16[m, k] with row stride x_ld (elements, >= k); y [m, n] contiguous,
 * y_dtype FH_BF16 (RNE of the fp32 sum, the reference's output rounding) or
 * FH_F32 (the fp32 sum itself). m <= 8 runs the decode GEMV, larger m the
 * prefill GEMM. m may be 0. */
int fh_q4_matmul(fh_device *dev, const uint16_t *x, int64_t m, int64_t k,
                 int64_t x_ld, const uint32_t *wq, const uint16_t *scales,
                 const uint16_t *biases, int64_t n, int64_t group, void *y,
                 int y_dtype);

/* Materialised dequantisation: out bf16[rows, k] = RNE_bf16(w). Bit-exact.
 * The value the prefill GEMM feeds to the matrix cores. */
int fh_q4_dequant(fh_device *dev, const uint32_t *wq, const uint16_t *scales,
                  const uint16_t *biases, int64_t rows, int64_t k, int64_t group,
                  uint16_t *out);

/* ======================================================================
 * Strided ops: the reference's non-quantized Ops (src/nn/primitive.rs:48-68)
 * over strided views, so that a backend can run every Op of the unchanged
 * model code (Device::run and Device::run_in_place, src/metal/mod.rs:639-
 * 725). Each entry point is one plain kernel of the Metal kernel it replaces
 * (src/metal/kernels/{copy,unary,binary,reduce,matmul,index_select,
 * slice_scatter}.metal) with the same arithmetic: fp32 math on values
 * decoded from the dtype, the output rounded once (RNE for bf16).
 *
 * A view is the reference's Layout flattened as StridedArgs is
 * (src/metal/args.rs:22-29): element offset, rank 0..4, sizes and strides in
 * elements (strides >= 0; a broadcast dim has stride 0). The pointer passed
 * beside a view is the storage base; the view addresses base + offset + sum
 * i_d * stride_d. Every element a view addresses must lie in one live
 * allocation of the device. Outputs are fresh and contiguous, as
 * Device::run returns them; shape rules are those of primitive::output
 * (src/nn/primitive.rs:146-289). dtype is an fh_dtype.
 * ====================================================================== */

typedef struct fh_view {
    int64_t offset;
    int32_t ndim;
    int64_t dims[4];
    int64_t strides[4];
} fh_view;

/* UnaryOp, BinaryOp, ReduceOp (src/nn/primitive.rs:14-46) */
typedef enum fh_unary_op { FH_NEG = 0, FH_EXP = 1, FH_SQRT = 2, FH_RECIPROCAL = 3 } fh_unary_op;
typedef enum fh_binary_op { FH_ADD = 0, FH_SUB = 1, FH_MUL = 2, FH_DIV = 3 } fh_binary_op;
typedef enum fh_reduce_op { FH_SUM = 0, FH_AMAX = 1, FH_ARGMAX = 2 } fh_reduce_op;

/* Op::Copy (copy_strided, copy.metal:1-13): dst = the view's elements in
 * row-major order. Any dtype. */
int fh_copy_strided(fh_device *dev, int dtype, const void *src, const fh_view *view, void *dst);

/* Op::ToDtype (to_dtype_strided, copy.metal:15-36): F32 <-> BF16 (RNE with
 * the quiet-NaN rule); the same float dtype is a copy. */
int fh_to_dtype(fh_device *dev, int from, const void *src, const fh_view *view, int to, void *dst);

/* Op::Unary (unary_strided, unary.metal:1-40) on F32 or BF16. */
int fh_unary(fh_device *dev, int op, int dtype, const void *src, const fh_view *view, void *dst);

/* Op::Binary (binary_strided, binary.metal:1-44). Both views have the
 * output's dims: a caller broadcasts first by expanding (stride 0), as
 * Tensor::binary does (src/nn/tensor.rs:332-343). */
int fh_binary(fh_device *dev, int op, int dtype, const void *lhs, const fh_view *lhs_view,
              const void *rhs, const fh_view *rhs_view, void *dst);

/* Op::Reduce{op, dim} (reduce_rows / argmax_rows, reduce.metal:1-93): one
 * block of 256 threads per output element; thread t folds k = t, t + 256,
 * ..., then a halving tree, the reference's order (its sums are bit-equal).
 * Output dims = the view's with dims[dim] = 1, contiguous; SUM/AMAX keep the
 * dtype, ARGMAX writes u32 (first index on ties). AMAX/ARGMAX over an empty
 * dim are refused (TensorError::EmptyReduction); an empty SUM is 0. */
int fh_reduce(fh_device *dev, int op, int dtype, const void *src, const fh_view *view, int32_t dim,
              void *dst);

/* Op::Matmul (MetalDevice::matmul, src/metal/mod.rs:434-481; matmul_tiled,
 * matmul.metal:29-65): lhs [..., m, k] x rhs [..., k, n] with equal batch
 * dims, out [..., m, n]; fp32 sums in order of k, output rounded once.
 * Any strides are read in place (no operand copy). */
int fh_matmul(fh_device *dev, int dtype, const void *lhs, const fh_view *lhs_view, const void *rhs,
              const fh_view *rhs_view, void *dst);

/* Op::IndexSelect{dim 0} (index_select_rows, index_select.metal:11-29):
 * table 2-D [rows, cols] (F32 or BF16), ids U32 1-D [n] -> dst [n, cols];
 * an id >= rows gives a zero row. */
int fh_index_select(fh_device *dev, int dtype, const void *table, const fh_view *table_view,
                    const uint32_t *ids, const fh_view *ids_view, void *dst);

/* Op::Cat{dim} (MetalDevice::cat, src/metal/mod.rs:502-524): dst = lhs then
 * rhs along dim; all other dims equal. */
int fh_cat(fh_device *dev, int dtype, int32_t dim, const void *lhs, const fh_view *lhs_view,
           const void *rhs, const fh_view *rhs_view, void *dst);

/* Device::run_in_place(Op::SliceScatter{dim, start}) (src/metal/mod.rs:697-
 * 725; slice_scatter_strided, slice_scatter.metal:1-21): writes src into
 * target[..., start : start + src.dims[dim], ...] in place. The target view
 * is contiguous (Tensor::slice_scatter requires it, src/nn/tensor.rs:
 * 307-316) and src may be strided. */
int fh_slice_scatter(fh_device *dev, int dtype, int32_t dim, int64_t start, void *target,
                     const fh_view *target_view, const void *src, const fh_view *src_view);

/* ======================================================================
 * Decoder-step ops: the plumbing around the q4 linears that a Llama decode
 * step needs, each one kernel where the reference runs several dispatches.
 * All tensors are bf16 (uint16_t bits) unless stated; every op rounds where
 * the reference's op sequence rounds (its tensors are bf16).
 * `positions` are device u32 arrays, so a captured decode step can be
 * replayed with the position advanced on the device (fh_advance_positions).
 * ====================================================================== */

/* RmsNorm::forward (src/nn/norm.rs:32-50), optionally fused with the
 * residual add before it (src/models/llama/model.rs:254-279):
 *   h = residual ? RNE(x + residual) : x   (h written to residual_out)
 *   y = RNE(RNE(h * 1/sqrt(sum(h^2)/dim + eps)) * weight)
 * x, residual, residual_out, y: [rows, dim]; weight: [dim]. dim is a multiple
 * of 8, at most 8192; operands are 16-byte aligned. residual_out may alias
 * residual (an in-place residual stream). */
int fh_rms_norm(fh_device *dev, const uint16_t *x, const uint16_t *residual,
                uint16_t *residual_out, const uint16_t *weight, int64_t rows, int64_t dim,
                float eps, uint16_t *y);

/* KV caches of the attention entry points below. One (sequence, KV head)
 * owns max_len * head_dim elements of each cache. V is [max_len][head_dim].
 * K holds the same keys in groups of 16: group g (keys 16 g .. 16 g + n_g -
 * 1, n_g = min(16, max_len - 16 g)) is n_g * head_dim contiguous elements
 * laid out [head_dim / 32][n_g][32], i.e. dim d of key j is element
 * 16 g * head_dim + (d / 32) * n_g * 32 + (j % 16) * 32 + d % 32 of the
 * region. The reference's StaticCache (src/nn/kv_cache.rs:41-80) keeps K as
 * [max_len][head_dim]; the regrouping lets a matrix-core fragment of 16 keys
 * x 32 dims be read as one 1 KB run. Sizes are unchanged. */

/* apply_rotary_pos_emb (src/models/llama/rotary_emb.rs:62-85) on q and k of
 * each token, then StaticCache::update (src/nn/kv_cache.rs:41-80) of k and v
 * at the token's position. qkv: [tokens, (n_heads + 2 n_kv) * head_dim] (q
 * heads, then k heads, then v heads); cos_tab/sin_tab: [table_len, head_dim];
 * positions: device u32 [tokens]; k_cache/v_cache: n_kv regions of max_len *
 * head_dim (K grouped as above); q_out: [tokens, n_heads, head_dim]. head_dim is a multiple of 16 and every
 * operand 16-byte aligned. A position >= max_len or >= table_len writes
 * nothing. */
int fh_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads,
               int64_t n_kv, int64_t head_dim, const uint16_t *cos_tab, const uint16_t *sin_tab,
               int64_t table_len, const uint32_t *positions, uint16_t *k_cache,
               uint16_t *v_cache, int64_t max_len, uint16_t *q_out);

/* Bytes of device workspace fh_attention needs for these sizes (the scores
 * and per-chunk softmax statistics of every row). */
int fh_attention_workspace(int64_t tokens, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                           int64_t max_len, uint64_t *bytes);

/* scaled_dot_product_attention (src/nn/attention.rs:23-60) with the causal
 * mask (src/nn/masking.rs:11-32): query token t attends keys 0..positions[t]
 * of its KV head (grouped-query: head h uses KV head h / (n_heads/n_kv)).
 * Scores RNE(q.k) (fp32 sums), times scale in fp32, softmax in fp32,
 * probabilities RNE to bf16 from the row's global max and sum, out =
 * RNE(sum p v). q, out: [tokens, n_heads * head_dim]; caches: n_kv regions of
 * max_len * head_dim (K grouped as above). head_dim is 64, 128 or 256 and n_heads/n_kv at most 8; tokens at
 * most 65535. The context is split into chunks of 64 keys scored in
 * parallel, and P.V is split over head_dim, so a long context fills the
 * device. workspace: at least fh_attention_workspace() bytes of device
 * memory, 16-byte aligned, no initial contents; calls that share a workspace
 * must not run concurrently. */
int fh_attention(fh_device *dev, const uint16_t *q, const uint16_t *k_cache,
                 const uint16_t *v_cache, const uint32_t *positions, int64_t tokens,
                 int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t max_len, float scale,
                 void *workspace, uint64_t workspace_bytes, uint16_t *out);

/* Bytes of device workspace fh_decode_attention needs for these sizes. */
int fh_decode_attention_workspace(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                  int64_t max_len, uint64_t *bytes);

/* The decode step's attention for a batch of sequences that each add one
 * token: fh_rope_kv's RoPE of the token's q and k and its cache write at
 * positions[b], then fh_attention over keys 0..positions[b] of sequence b --
 * the same rounding points, in two or three kernel launches, or in one for
 * few rows with max_len <= 1024 and head_dim 64 or 128 (the workspace is then
 * not touched, but is still checked and required). qkv:
 * [batch, (n_heads + 2 n_kv) * head_dim]; cos_tab/sin_tab: [table_len,
 * head_dim]; positions: device u32 [batch]; k_cache/v_cache: batch x n_kv
 * regions of max_len * head_dim (one cache per sequence, K grouped as above);
 * out: [batch, n_heads *
 * head_dim]. A position >= max_len or >= table_len writes nothing to the
 * caches and zeros to out. head_dim is 64, 128 or 256, n_heads/n_kv at most
 * 8, batch at most 65535, operands 16-byte aligned. workspace: as for
 * fh_attention, at least fh_decode_attention_workspace() bytes. */
int fh_decode_attention(fh_device *dev, const uint16_t *qkv, int64_t batch, int64_t n_heads,
                        int64_t n_kv, int64_t head_dim, const uint16_t *cos_tab,
                        const uint16_t *sin_tab, int64_t table_len, const uint32_t *positions,
                        uint16_t *k_cache, uint16_t *v_cache, int64_t max_len, float scale,
                        void *workspace, uint64_t workspace_bytes, uint16_t *out);

/* fh_decode_attention without a workspace argument, for callers that cannot
 * allocate (code under graph capture, tight serving loops, harnesses that
 * forbid allocation). No counterpart in the reference. The workspace is a
 * static array of FH_DECODE_SCRATCH_BYTES in device memory, one per GPU,
 * held from the library's first use on that GPU until the process ends; this
 * call allocates nothing (on a profiled device it records only pooled
 * events). Sizes whose workspace (fh_decode_attention_workspace) exceeds it
 * return FH_ERR_UNSUPPORTED. Every call on one GPU shares the array: calls
 * that overlap on one GPU (from two fh_devices' streams) race. The workspace
 * needs no initial contents, so nothing is cleared between calls. */
#define FH_DECODE_SCRATCH_BYTES (32ull << 20)
int fh_decode_attention_noalloc(fh_device *dev, const uint16_t *qkv, int64_t batch, int64_t n_heads,
                                int64_t n_kv, int64_t head_dim, const uint16_t *cos_tab,
                                const uint16_t *sin_tab, int64_t table_len, const uint32_t *positions,
                                uint16_t *k_cache, uint16_t *v_cache, int64_t max_len, float scale,
                                uint16_t *out);

/* Decode-step fusions of the q4 Linear (m <= 8 rows, the GEMV; larger m
 * returns FH_ERR_UNSUPPORTED -- use the unfused ops -- except
 * fh_q4_gate_up_silu without a norm weight, below). Same arithmetic as the
 * unfused sequence, with no intermediate tensor in memory:
 *   fh_q4_matmul_rmsnorm: y = fh_rms_norm(x, residual, residual_out,
 *     norm_weight, eps) @ W^T (src/nn/norm.rs:32-50 then src/nn/linear.rs:
 *     22-35). x, residual, residual_out: [m, k] (row stride k); residual and
 *     residual_out may be null; residual_out (the updated residual stream h)
 *     must not overlap x or residual. The sum of squares runs in another
 *     order than fh_rms_norm's (a normalised value can differ by one bf16 ulp).
 *   fh_q4_gate_up_silu: act = fh_silu_mul(x' @ W^T) for W = [gate; up] rows
 *     (n = 2f): act[:, j] = RNE(RNE(g_j / (exp(-g_j) + 1)) * u_j) with g, u
 *     the bf16 outputs of the linear (src/models/llama/mlp.rs:49-58); act:
 *     [m, f] bf16. x' = x, or with norm_weight, the RMSNorm above (residual
 *     arguments as for fh_q4_matmul_rmsnorm). Above 8 rows, without a norm
 *     weight or residual: the prompt GEMM with the activation in its
 *     epilogue (few rows: the GEMM, its sums in the device's partial area, and
 *     the activation), when its tiles of 256 rows x 128 gate/up pairs fill the
 *     GPU (f % 128 == 0, k % 512 == 0; x and act 16-byte aligned, act not
 *     overlapping x); other shapes return FH_ERR_UNSUPPORTED. Bit-identical
 *     to fh_q4_matmul then fh_silu_mul.
 * The q4 operands follow fh_q4_matmul (group 64); x 16-byte aligned. */
int fh_q4_matmul_rmsnorm(fh_device *dev, const uint16_t *x, const uint16_t *residual,
                         uint16_t *residual_out, const uint16_t *norm_weight, float eps, int64_t m,
                         int64_t k, const uint32_t *wq, const uint16_t *scales,
                         const uint16_t *biases, int64_t n, int64_t group, void *y, int y_dtype);
int fh_q4_gate_up_silu(fh_device *dev, const uint16_t *x, const uint16_t *residual,
                       uint16_t *residual_out, const uint16_t *norm_weight, float eps, int64_t m,
                       int64_t k, const uint32_t *wq, const uint16_t *scales, const uint16_t *biases,
                       int64_t n, int64_t group, uint16_t *act);

/* A load-time copy of a q4 weight's scales and biases, interleaved per group
 * pair: sb (u32 [n, k / 64], 16-byte aligned) gets at dword 2p of row r the
 * scales of groups 2p and 2p + 1 (group 2p in the low half) and at dword
 * 2p + 1 their biases. fh_q4_weight.sb takes it; the 2..8-row decode GEMV of
 * fh_llama_forward then reads a chunk's scales and biases with one load
 * instead of two (the same values: results are unchanged). No counterpart in
 * the reference (its Linear reads the separate scales / biases tensors,
 * src/nn/linear.rs:22-35); a data layout of this library's decoder.
 * group = 64, k a multiple of 128. */
int fh_q4_interleave(fh_device *dev, const uint16_t *scales, const uint16_t *biases, int64_t n,
                     int64_t k, int64_t group, uint32_t *sb);

/* A load-time copy of a q4 weight's packed words in the batched decode
 * GEMV's task order: wt (u32, n * k / 8 words, 16-byte aligned) holds, for
 * task tile t, group pair p and column c < 16, the 16 words of pair p of
 * weight row r(t, c) at words ((t * k / 128 + p) * 16 + c) * 16. r(t, c) =
 * 16 t + c, or with silu_pairs (a [gate; up] weight of n = 2f rows) the gate
 * row 8 t + c for c < 8 and the up row f + 8 t + c - 8. fh_q4_weight.wt
 * takes it (silu_pairs = 1 for the gate/up weight, 0 for the others); the
 * 2..8-row GEMVs of fh_llama_forward then read one contiguous KiB per
 * wavefront load instead of 16 rows x 64 bytes (the same values: results
 * are unchanged). No counterpart in the reference (its Linear reads the
 * packed tensor as stored, src/nn/linear.rs:22-35); a data layout of this
 * library's decoder. group = 64; n a multiple of 16 (32 with silu_pairs),
 * k of 128; wt must not overlap wq. */
int fh_q4_tile(fh_device *dev, const uint32_t *wq, int64_t n, int64_t k, int64_t group, int silu_pairs,
               uint32_t *wt);

/* LlamaMlp's act_fn(gate) * up (src/models/llama/mlp.rs:49-58, Silu at
 * src/nn/activation.rs:19-28): gate_up row = [gate (f) | up (f)],
 * out = RNE(RNE(g / (1 + exp(-g))) * u), out: [rows, f]. */
int fh_silu_mul(fh_device *dev, const uint16_t *gate_up, int64_t rows, int64_t f, uint16_t *out);

/* Greedy next token (src/generate/mod.rs:192-204): row argmax of bf16
 * values, ties to the lowest index (src/metal/kernels/reduce.metal:42-78).
 * x: [rows, n]; out: u32 [rows]. */
int fh_argmax(fh_device *dev, const uint16_t *x, int64_t rows, int64_t n, uint32_t *out);

/* For each sequence r < rows: log[r * capacity + position[r] - base] =
 * token[r] when 0 <= position[r] - base < capacity. The greedy loop's token
 * record (token_ids per batch row, src/bench/mod.rs:250-300), kept on the
 * device so a captured step can be replayed without reading back each
 * token. token, position: u32 [rows]; log: u32 [rows, capacity]. */
int fh_append_token(fh_device *dev, const uint32_t *token, int64_t rows, uint32_t *log,
                    const uint32_t *position, int64_t base, int64_t capacity);

/* positions[i] += by for i < n, on the device's stream. */
int fh_advance_positions(fh_device *dev, uint32_t *positions, int64_t n, int64_t by);

/* fh_append_token(dev, token, rows, log, position, base, capacity), then
 * fh_advance_positions(dev, position, rows, by), as one launch: the decode
 * step's token record and position bump (src/generate/mod.rs:45-90), one
 * dispatch fewer per replayed step. With capacity 0 nothing is logged and
 * log may be null. token and position may share memory. */
int fh_append_token_advance(fh_device *dev, const uint32_t *token, int64_t rows, uint32_t *log,
                            uint32_t *position, int64_t base, int64_t capacity, int64_t by);

/* ======================================================================
 * Serving many requests at once: a paged KV cache, low-rank adapters and
 * logit rules. No counterpart in the reference, which decodes equal-length
 * sequences over one static cache each (src/nn/kv_cache.rs:13-39), with one
 * set of weights, greedily. Unlike the decoder-step ops above, which round
 * where the reference's op sequence rounds, these keep every sum and the
 * softmax's maximum and sum in fp32 and round each output once; a factor that
 * they hold in fewer bits on the way is named at its call.
 *
 * A paged cache is a pool of n_pages pages of page_size tokens (a multiple of
 * 16). Page p of the K pool and of the V pool holds n_kv regions of page_size
 * * head_dim elements, each laid out as a cache of max_len = page_size (K
 * grouped by 16 keys, V [page_size][head_dim]); the pools are
 * [n_pages][n_kv][page_size * head_dim]. page_table (device u32 [n_seqs,
 * max_pages]) names sequence s's pages in order: position j of s is slot j %
 * page_size of page page_table[s * max_pages + j / page_size]. Entries behind
 * a sequence's last page are not read. Positions, sequences and page ids are
 * device data that the host cannot check: an entry that names no page
 * (>= n_pages) is left alone, as described for each call. max_pages *
 * page_size is at most 2^31 - 1; pools may pass 4 GiB. Pools and 2-byte
 * operands are 16-byte aligned, lists of 4-byte entries 4-byte aligned.
 * ====================================================================== */

/* apply_rotary_pos_emb on q and k of each token, then k and v written to the
 * token's place in the paged cache (fh_rope_kv for requests of any lengths, as
 * a packed batch of prompts or one new token each):
 *   q' = RNE(q * cos + rot(q) * sin), k' the same, v as it is.
 * qkv: [tokens, (n_heads + 2 n_kv) * head_dim]; cos_tab / sin_tab:
 * [table_len, head_dim]; sequences: u32 [tokens], or null where token t is of
 * sequence t (tokens <= n_seqs); positions: u32 [tokens]; q_out: [tokens,
 * n_heads, head_dim]. q_out and the pools overlap neither each other nor the
 * inputs. A token whose position is >= max_pages * page_size or >= table_len,
 * whose sequence is >= n_seqs or whose page is >= n_pages writes nothing,
 * neither to the pools nor to q_out (a padded row takes a position past the
 * pages, far enough below 2^32 where fh_advance_positions moves it on). Two
 * tokens of one sequence and position leave the values of either in each
 * 16-byte piece. head_dim is a multiple of 32, at most 256, tokens at most
 * 2^24 - 1. */
int fh_paged_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads,
                     int64_t n_kv, int64_t head_dim, const uint16_t *cos_tab,
                     const uint16_t *sin_tab, int64_t table_len, const uint32_t *sequences,
                     const uint32_t *positions, const uint32_t *page_table, int64_t n_seqs,
                     int64_t max_pages, uint16_t *k_pages, uint16_t *v_pages, int64_t n_pages,
                     int64_t page_size, uint16_t *q_out);

/* Bytes of device workspace fh_paged_attention needs for these sizes, never
 * less for a larger batch. */
int fh_paged_attention_workspace(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                 int64_t page_size, int64_t max_pages, uint64_t *bytes);

/* Attention of one new token of each sequence over the paged cache, whose
 * keys and values (the new token's among them) fh_paged_rope_kv has written:
 *   s_j = scale * (q . k_j), j = 0..positions[b],
 *   out[b] = RNE(sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s))
 * with fp32 sums; exp(..) as v's factor has 16 bits (off by 2^-16 of a term
 * at most). q, out: [batch, n_heads * head_dim]; row b of page_table and
 * positions[b] belong to sequence b; query head h uses KV head h / (n_heads /
 * n_kv). A sequence whose position is >= max_pages * page_size is idle: zeros
 * to its rows of out. Keys of a table entry that names no page are left out; a
 * sequence left with no key gets zeros. What lies in a page behind the
 * position is not used, whatever its bits. A row whose every score is -inf is
 * NaN. Up to 1024 sequences share the GPU by their lengths; in a larger batch
 * each has one block per KV head and 8 query heads, so a long one among them
 * is faster in a call of its own. head_dim is 64, 128 or 256; any n_heads /
 * n_kv; batch at most 65535, and batch * (max_pages * page_size / 128 + 1) at
 * most 2^31 - 1; out does not overlap the inputs. workspace: at least
 * fh_paged_attention_workspace() bytes, 16-byte aligned, no initial contents;
 * calls that share a workspace must not run concurrently. */
int fh_paged_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t n_heads,
                       int64_t n_kv, int64_t head_dim, const uint16_t *k_pages,
                       const uint16_t *v_pages, int64_t n_pages, int64_t page_size,
                       const uint32_t *page_table, int64_t max_pages, const uint32_t *positions,
                       float scale, void *workspace, uint64_t workspace_bytes, uint16_t *out);

/* Bytes of device workspace fh_lora_add needs for these sizes, never less for
 * more rows. */
int fh_lora_workspace(int64_t m, int64_t k, int64_t rank, uint64_t *bytes);

/* The low-rank adapters of many requests beside a shared projection (base,
 * what fh_q4_matmul gave for the same x):
 *   y[i, :] = RNE(base[i, :] + scales[a] * (x[i, :] . A_a^T) . B_a^T),
 *   a = adapters[i],
 * with fp32 sums; scales[a] * (x . A_a^T) as B's factor has 16 bits for bf16
 * results (off by 2^-16 of a term at most), 24 for f32. x: bf16 [m, k] with
 * row stride x_ld (a multiple of 8, >= k); a: bf16 [n_adapters, rank, k]; b:
 * bf16 [n_adapters, n, rank]; scales: f32 [n_adapters]; adapters: u32 [m], in
 * any order, a row of a value >= n_adapters taking no adapter (y = base
 * there). An adapter of a lower rank is filled up with zeros. base, y: [m, n]
 * of `dtype` (FH_BF16 or FH_F32) with row strides base_ld, y_ld >= n; y is
 * base itself (the same pointer and stride) or does not overlap the operands.
 * rank and k are multiples of 8, rank at most 128; n is any, m at most
 * 4194240; x, a, b 16-byte aligned. workspace: at least fh_lora_workspace()
 * bytes, 16-byte aligned, no initial contents; calls that share a workspace
 * must not run concurrently. */
int fh_lora_add(fh_device *dev, const uint16_t *x, int64_t m, int64_t k, int64_t x_ld,
                const uint16_t *a, const uint16_t *b, const float *scales, int64_t n_adapters,
                int64_t rank, int64_t n, const uint32_t *adapters, const void *base,
                int64_t base_ld, void *y, int64_t y_ld, int dtype, void *workspace,
                uint64_t workspace_bytes);

/* What fh_logits_process applies; every pointer is device memory, and each
 * rule whose pointer is null is left out. */
typedef struct fh_logit_rules {
    const uint32_t *history;     /* [rows, history_ld] token ids: the prompt, then what was generated */
    int64_t history_ld;
    const uint32_t *history_len; /* [rows] ids in use (at most history_ld are) */
    const uint32_t *prompt_len;  /* [rows] leading ids that are the prompt's; null: 0 */
    const float *repetition;     /* [rows] */
    const float *frequency;      /* [rows] */
    const float *presence;       /* [rows] */
    const uint32_t *bias_ids;    /* [rows, bias_ld] */
    const float *bias_values;    /* [rows, bias_ld] */
    int64_t bias_ld;
    const uint32_t *bias_len;    /* [rows] entries in use (at most bias_ld are); null: bias_ld */
    const uint32_t *mask;        /* [rows, ceil(n / 32)]: bit j % 32 of word j / 32 allows token j */
} fh_logit_rules;

/* Penalties for repeated tokens, biases and a grammar's mask on logits, before
 * fh_argmax. For token j of a row, c = its count among the generated ids:
 *   1. repetition, where j is among the history's ids: z = z > 0 ? z / r : z * r
 *   2. frequency and presence: z = (z - f * c) - (c > 0 ? p : 0)
 *   3. bias: z = z + value (an id listed twice: the last entry counts)
 *   4. mask: z = -inf where j's bit is 0, whatever z was
 * each step rounded to fp32, then z once to dtype. logits, out: [rows, n] of
 * `dtype` (FH_BF16 or FH_F32); out may be logits itself, else does not
 * overlap the inputs. An id >= n is passed over. history and history_len go
 * together (the three penalties need them), as do bias_ids and bias_values.
 * rows is at most 65535. */
int fh_logits_process(fh_device *dev, const void *logits, int dtype, int64_t rows, int64_t n,
                      const fh_logit_rules *rules, void *out);

/* ======================================================================
 * Drafting several tokens ahead: each step runs a tree of drafted tokens (or a
 * chain) through the model at once and keeps the branch that the target's
 * distributions accept. No counterpart in the reference, which decodes one
 * token at a time (src/generate/mod.rs:150-204). A sequence b with lengths[b]
 * tokens in the paged cache above has its tree's nodes at the places lengths[b]
 * + 0, 1, ..: node 0, the root, is the last token emitted, whose key and value
 * the cache does not hold yet; a node's parent comes before it. What holds for
 * the serving calls above (device data that names nothing, alignment, sums in
 * fp32, one rounding of each output) holds here. A step is
 *   fh_paged_reserve        pages for the nodes
 *   fh_paged_norm_rope_kv   each layer's k and v of the nodes, at their places
 *   fh_paged_tree_attention each layer's attention of the nodes
 *   fh_logits_probs         the distribution behind each node
 *   fh_verify_draft         the accepted path and the token after it
 *   fh_paged_compact        the path's keys and values to the front, new lengths
 * and may be captured as a whole.
 * ====================================================================== */

/* fh_paged_rope_kv with a norm of each q and k head before the rotation and
 * places apart from the positions:
 *   q' = RNE(n * cos + rot(n) * sin), n = q * w / sqrt(sum(q^2) / head_dim + eps),
 * w = q_norm for q's heads, k_norm for k's (bf16 [head_dim]; null: n = q, n =
 * k); v as it is. The sum of squares, n and the rotation are fp32: squares past
 * fp32's largest make n zero, those below its smallest count as 0 (with eps 0 a
 * head of nothing else has no finite n). positions (u32 [tokens]) give the rotation,
 * slots (u32 [tokens], null: the positions) the place in the sequence: the nodes
 * of a tree share positions. A token whose position is >= table_len, whose slot
 * is >= max_pages * page_size, whose sequence is >= n_seqs or whose page is >=
 * n_pages writes nothing. eps >= 0; the rest is as for fh_paged_rope_kv. */
int fh_paged_norm_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads,
                          int64_t n_kv, int64_t head_dim, const uint16_t *q_norm,
                          const uint16_t *k_norm, float eps, const uint16_t *cos_tab,
                          const uint16_t *sin_tab, int64_t table_len, const uint32_t *sequences,
                          const uint32_t *positions, const uint32_t *slots,
                          const uint32_t *page_table, int64_t n_seqs, int64_t max_pages,
                          uint16_t *k_pages, uint16_t *v_pages, int64_t n_pages, int64_t page_size,
                          uint16_t *q_out);

/* Bytes of device workspace fh_paged_tree_attention needs for these sizes,
 * never less for a larger batch. */
int fh_paged_tree_attention_workspace(int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv,
                                      int64_t head_dim, int64_t page_size, int64_t max_pages,
                                      uint64_t *bytes);

/* Attention of each sequence's nodes over its cached tokens and its tree (keys
 * and values of both are in the paged cache): node i of sequence b sees keys 0
 * .. lengths[b] - 1, and key lengths[b] + j for each j < counts[b] whose bit (bit
 * j % 32 of word j / 32) in masks[b, i] is set, whether that is i itself or not:
 *   s_j = scale * (q . k_j), out[b, i] = RNE(sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s))
 * q, out: [batch, width, n_heads * head_dim]; lengths: u32 [batch]; counts: u32
 * [batch], nodes in use (more than width count as width; null: width); masks:
 * u32 [batch, width, ceil(width / 32)], or null for chains (node i sees nodes 0
 * .. i). A row past a sequence's nodes, one that sees no key and those of a
 * sequence whose nodes do not fit its table (lengths[b] + counts[b] > max_pages
 * * page_size: idle) are zeros. Keys of a table entry that names no page are
 * left out. What lies at places that a row does not see is not used for it,
 * whatever its bits. A row whose every score is -inf is NaN; one of finite scores
 * and values is finite, however large they are (beside sums past 2^64, values below
 * 2^-78 may count as 0). exp(..) as v's factor has 16 bits (off by 2^-16 of a term
 * at most). head_dim is 64, 128 or 256, any n_heads / n_kv; width is 1 to 1024,
 * batch at most 65535, scale above 0 and at most 2e38; out does not overlap the
 * inputs. workspace: as for fh_paged_attention, at least
 * fh_paged_tree_attention_workspace() bytes. */
int fh_paged_tree_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t width,
                            int64_t n_heads, int64_t n_kv, int64_t head_dim,
                            const uint16_t *k_pages, const uint16_t *v_pages, int64_t n_pages,
                            int64_t page_size, const uint32_t *page_table, int64_t max_pages,
                            const uint32_t *lengths, const uint32_t *counts, const uint32_t *masks,
                            float scale, void *workspace, uint64_t workspace_bytes, uint16_t *out);

/* Bytes of device workspace fh_logits_probs needs for these sizes, never less
 * for more rows. */
int fh_logits_probs_workspace(int64_t rows, int64_t n, uint64_t *bytes);

/* The distribution of each row of logits at its temperature:
 *   probs[r, j] = exp((z_j - max z) / t) / sum_j exp((z_j - max z) / t), t = temperatures[r]
 * logits: [rows, n] of `dtype` (FH_BF16 or FH_F32); temperatures: f32 [rows],
 * null for 1. A temperature that is not above 0 is a greedy request's: 1 at the
 * row's largest logit (the first of equals), 0 elsewhere. Others count as at
 * least 1e-30 and at most 1e30. A NaN counts as -inf; infinite logits share a
 * row evenly; a row of nothing but -inf is zeros. probs: f32 [rows, n], does not
 * overlap the inputs. rows is at most 65535. workspace: at least
 * fh_logits_probs_workspace() bytes, 16-byte aligned, no initial contents;
 * calls that share a workspace must not run concurrently. */
int fh_logits_probs(fh_device *dev, const void *logits, int dtype, int64_t rows, int64_t n,
                    const float *temperatures, void *workspace, uint64_t workspace_bytes,
                    float *probs);

/* Bytes of device workspace fh_verify_draft needs for these sizes, never less
 * for a larger batch. */
int fh_verify_draft_workspace(int64_t batch, int64_t width, int64_t n, uint64_t *bytes);

/* Which of a tree's drafted tokens the target's distributions accept, and the
 * token after them, so that what is emitted is distributed as the target alone
 * would have it. probs: f32 [batch, width, n], row i the target's distribution
 * behind node i; draft_probs: the same of the draft model, row i what node i's
 * children were drawn from, or null where the drafted tokens were picked without
 * chance (then q below is 1 at the child's token, 0 elsewhere). tokens, parents:
 * u32 [batch, width], node i's token and parent (parents null: i - 1; node 0 has
 * none, tokens[b, 0] is not read); counts: u32 [batch], nodes in use (more than
 * width count as width; null: width); uniforms: f32 [batch, width] in [0, 1).
 *   Start at node a = 0 with w = probs[a], Z = 1. Its children are asked in order:
 *   child i of token x is accepted if uniforms[i] * q(x) * Z < w(x): go on from a = i.
 *   Else w becomes max(w - Z q, 0) and Z its sum (q at x alone: w(x) becomes 0, and Z
 *   is less by what it was).
 *   When no child is left, the first token whose running sum of w is past uniforms[0]
 *   times w's sum follows (w = probs[a] again where nothing was left of it).
 * path (u32 [batch, width]) gets the accepted nodes, the root first, accepted
 * (u32 [batch]) their number, out_tokens (u32 [batch, width]) their tokens
 * without the root's, then the one that follows; 0xFFFFFFFF behind them, and in
 * place of a token that follows a row without any positive entry. A sequence of
 * no nodes accepts 0. Sums and comparisons are fp64; entries of probs that are
 * not above 0 count as 0; no entry of either is infinite, none of draft_probs
 * negative or NaN (a sequence with one may get any token below n, or
 * 0xFFFFFFFF). A child whose token is >= n, or whose
 * parent does not come before it, is passed over. With width 1 this draws
 * a token of each row. width is 1 to 1024, batch at most 65535; no output
 * overlaps an input or another. workspace: at least fh_verify_draft_workspace()
 * bytes, 16-byte aligned, no initial contents; calls that share a workspace must
 * not run concurrently. */
int fh_verify_draft(fh_device *dev, const float *probs, const float *draft_probs, int64_t batch,
                    int64_t width, int64_t n, const uint32_t *tokens, const uint32_t *parents,
                    const uint32_t *counts, const float *uniforms, void *workspace,
                    uint64_t workspace_bytes, uint32_t *path, uint32_t *out_tokens,
                    uint32_t *accepted);

/* One layer's pools of a paged cache. */
typedef struct fh_paged_pool {
    uint16_t *k_pages;
    uint16_t *v_pages;
} fh_paged_pool;

/* A paged cache of all layers, for the calls below: pools is a host array of
 * n_layers entries (at most 128), which share the page table; page_table (u32
 * [n_seqs, max_pages]), lengths (u32 [n_seqs], tokens of each sequence) and refs
 * (u32 [n_pages], how many table entries name each page; 0: the page is free)
 * are device memory. No two of them overlap. Entries of a row that hold no page
 * name none (0xFFFFFFFF). n_seqs is at most 16384. */
typedef struct fh_paged_cache {
    const fh_paged_pool *pools;
    int64_t n_layers, n_kv, head_dim, n_pages, page_size;
    uint32_t *page_table;
    int64_t n_seqs, max_pages;
    uint32_t *lengths;
    uint32_t *refs;
} fh_paged_cache;

/* Pages for the next extra[s] tokens of each sequence: the table entries of
 * places lengths[s] .. lengths[s] + extra[s] - 1 that name no page get the lowest
 * free pages, by sequence, then by entry; their refs become 1. missing (u32
 * [n_seqs], or null) gets how many entries of a sequence got none, since the
 * table or the free pages ended. At most 16384 pages are handed out in a call.
 * extra: u32 [n_seqs]. pools and n_layers are not used, and pools may be null. */
int fh_paged_reserve(fh_device *dev, const fh_paged_cache *cache, const uint32_t *extra,
                     uint32_t *missing);

/* Makes sequence to[i] a copy of sequence from[i], for i < n: to's own pages are
 * freed, from's whole pages shared, and the tokens of its last page, if that is
 * not full, copied in every layer to the lowest free page (forks in order).
 * lengths[to] = lengths[from]; pages past from's length stay its own. lost (u32
 * [n]) gets 1 where no page was free (to is then empty) or the fork was passed
 * over and changed nothing: from[i] or to[i] >= n_seqs, to[i] among from or
 * among the entries of to before i, or a length past the table; else 0. from,
 * to: u32 [n], n at most 1024. */
int fh_paged_fork(fh_device *dev, const fh_paged_cache *cache, const uint32_t *from,
                  const uint32_t *to, int64_t n, uint32_t *lost);

/* Empties the sequences seqs[i], i < n (u32 [n]; >= n_seqs: passed over): the refs
 * of their pages are one less, their table entries name no page, their lengths
 * are 0. A sequence named twice is emptied once. n is at most 65535. pools and
 * n_layers are not used, and pools may be null. */
int fh_paged_free(fh_device *dev, const fh_paged_cache *cache, const uint32_t *seqs, int64_t n);

/* Moves an accepted path's keys and values to the front of its tree, in every
 * layer: place lengths[s] + i takes what is at lengths[s] + path[s, i], for i <
 * accepted[s] (at most width), as fh_verify_draft gives them: path[s, i] is
 * at least i and rises with i (of other paths a place may get another node's
 * values). Places past the table or without a page are passed over.
 * new_lengths[s] = lengths[s] + accepted[s]; it is lengths itself (one launch
 * more) or overlaps nothing. path: u32 [n_seqs, width]; accepted: u32 [n_seqs].
 * refs is not used, and may be null; a place's page is one sequence's alone, as
 * fh_paged_fork leaves them. */
int fh_paged_compact(fh_device *dev, const fh_paged_cache *cache, const uint32_t *path,
                     const uint32_t *accepted, int64_t width, uint32_t *new_lengths);

/* ======================================================================
 * The decoder forward issued from native code: the layer loop that a
 * caller would otherwise drive op by op, so an eager prefill is not bound
 * by per-call host overhead.
 * ====================================================================== */

/* A q4 weight: n rows of k columns (group 64), as fh_q4_matmul takes it.
 * sb: null, or fh_q4_interleave's copy of scales / biases, which the
 * batched decode GEMVs (2..8 rows) then read instead. wt: null, or (with sb)
 * fh_q4_tile's copy of the words, built with silu_pairs = 1 for gate_up and
 * 0 for the other weights, which the batched decode GEMVs read instead of
 * wq. */
typedef struct fh_q4_weight {
    const uint32_t *wq;
    const uint16_t *scales;
    const uint16_t *biases;
    int64_t n;
    int64_t k;
    const uint32_t *sb;
    const uint32_t *wt;
} fh_q4_weight;

/* One decoder layer (LlamaDecoderLayer, src/models/llama/model.rs:47, :254-280):
 * qkv = [Wq; Wk; Wv] and gate_up = [Wgate; Wup] rows; bf16 norm weights
 * [hidden]; caches: batch x n_kv regions of max_len * head_dim (K grouped
 * as for fh_rope_kv). */
typedef struct fh_llama_layer {
    fh_q4_weight qkv, o, gate_up, down;
    const uint16_t *input_norm;
    const uint16_t *post_norm;
    uint16_t *k_cache;
    uint16_t *v_cache;
} fh_llama_layer;

/* A Llama model on one device and the buffers of one forward. rows =
 * batch * max_tokens: h, h2, x, o [rows, hidden]; qkv [rows, (n_heads +
 * 2 n_kv) * head_dim]; q, attn [rows, n_heads * head_dim]; gate_up
 * [rows, 2 ffn]; act [rows, ffn]; logits [batch, vocab]. cos_tab/sin_tab:
 * [max_len, head_dim]. Workspaces: at least fh_attention_workspace(
 * max_tokens, ...) and fh_decode_attention_workspace(batch, ...) bytes.
 * `layers` is a host array of n_layers entries. */
typedef struct fh_llama_model {
    int64_t n_layers, hidden, n_heads, n_kv_heads, head_dim, ffn, vocab;
    int64_t batch, max_len, max_tokens;
    float rms_norm_eps;
    float scale;
    const fh_llama_layer *layers;
    fh_q4_weight embed;
    const uint16_t *final_norm;
    const uint16_t *cos_tab;
    const uint16_t *sin_tab;
    uint16_t *h, *h2, *x, *qkv, *q, *attn, *o, *gate_up, *act, *logits;
    void *attn_workspace;
    uint64_t attn_workspace_bytes;
    void *decode_workspace;
    uint64_t decode_workspace_bytes;
} fh_llama_model;

/* LlamaModel::forward (src/models/llama/model.rs:92-121) and the greedy
 * pick of Decoder::step (src/generate/mod.rs:150-204): ids and positions
 * (device u32 [batch, seq_tokens], sequence-major) run through the embedding,
 * every layer and the tied LM head of each sequence's last row; next (device
 * u32 [batch]) gets each sequence's argmax. The same op sequence as calling
 * the ops above one by one: up to 8 rows the RMSNorms, residual adds and SiLU
 * go inside the GEMVs and one new token's RoPE and cache write inside
 * fh_decode_attention; above 8 rows the unfused ops run, and prefill
 * attention gives what fh_attention gives for each sequence alone. Above 8 rows a GEMM that splits K
 * passes its f32 partials (the device's partial area) to the RoPE, RMSNorm
 * or SiLU after it, which adds them in the order of the GEMM's own reduce:
 * the results are bit-identical to the op sequence, but the buffers o,
 * gate_up and (seq_tokens > 1) qkv are then not written. The weight shapes
 * are checked against the config before any work is issued; every op checks
 * its own ranges as it runs. May be captured (fh_capture_begin).
 * 1 <= seq_tokens <= max_tokens. */
int fh_llama_forward(fh_device *dev, const fh_llama_model *model, int64_t seq_tokens,
                     const uint32_t *ids, const uint32_t *positions, uint32_t *next);

#ifdef __cplusplus
}
#endif

#endif
