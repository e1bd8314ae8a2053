/*
 * mfcuda.h -- C ABI of the B200 (sm_100a) backend for manifesto's
 * data-parallel hot path: dtype conversion, packed Int4 group dequant,
 * axpy / scalar-broadcast vector loops, fused elementwise chains and
 * per-tensor amax-scaled FP8 quantisation (single tensor and whole
 * checkpoints sharded over several GPUs), and a decoding step over a paged
 * key-value cache (page tables, rotary positions, cache writes, attention).
 *
 * Conventions
 *   - Plain C types only: pointers, int32_t/int64_t/size_t, float.
 *   - Every entry point returns an int status: MF_OK (0) or a negative
 *     MF_ERR_* code. Each negative code corresponds 1:1 to a sentinel in
 *     manifesto tensor/errors.go:10-72 (see the table beside the enum), so
 *     a cgo adapter maps them with a switch. The message of the most recent
 *     failure on the calling OS thread is available from mf_last_error().
 *   - Device pointers are plain CUDA device addresses on the device chosen
 *     with mf_init(). Stream and event handles are cudaStream_t / cudaEvent_t
 *     cast to void*; a NULL stream is the legacy default stream.
 *   - No entry point synchronises the host with the device except the ones
 *     whose name says so (mf_stream_sync, mf_event_sync, mf_device_sync) and
 *     the set-up calls (mf_init, mf_alloc, mf_free, mf_fused_compile,
 *     mf_comm_init, mf_paged_attn_create, mf_paged_attn_destroy). Scalar
 *     results such as amax are written to device memory, never returned to the
 *     host (manifesto scripts/check_banned.sh:28-40 forbids host syncs on the
 *     launch path).
 *   - Arithmetic follows manifesto's Go scalar code bit for bit, including
 *     its FP8 rounding quirks (compat = MF_COMPAT_REFERENCE). The file:line
 *     each entry point replaces is given in its comment; paths are inside
 *     the manifesto Go module.
 */
#ifndef MFCUDA_H
#define MFCUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MFCUDA_ABI_VERSION 1

/* ---------------------------------------------------------------------
 * dtype wire codes: identical to dtype.DType (dtype/dtype.go:29-49).
 * ------------------------------------------------------------------- */
enum mf_dtype {
    MF_DT_INVALID = 0,
    MF_DT_F64 = 1,
    MF_DT_F32 = 2,
    MF_DT_F16 = 3,
    MF_DT_BF16 = 4,
    MF_DT_F8E4M3 = 5,
    MF_DT_F8E5M2 = 6,
    MF_DT_I64 = 7,
    MF_DT_I32 = 8,
    MF_DT_I16 = 9,
    MF_DT_I8 = 10,
    MF_DT_I4 = 11, /* packed two per byte, element 2i in the low nibble */
    MF_DT_U64 = 12,
    MF_DT_U32 = 13,
    MF_DT_U16 = 14,
    MF_DT_U8 = 15
};

/* ---------------------------------------------------------------------
 * Status codes.  Negative values map onto tensor/errors.go sentinels:
 *   MF_ERR_DTYPE_MISMATCH       -> tensor.ErrDTypeMismatch       (:13)
 *   MF_ERR_DTYPE_UNSUPPORTED    -> tensor.ErrDTypeUnsupported    (:18)
 *   MF_ERR_LAYOUT_UNSUPPORTED   -> tensor.ErrLayoutUnsupported   (:23)
 *   MF_ERR_SHAPE_MISMATCH       -> tensor.ErrShapeMismatch       (:28)
 *   MF_ERR_BACKEND_CLOSED       -> tensor.ErrBackendClosed       (:46)
 *   MF_ERR_SHAPE_INVALID        -> tensor.ErrShapeInvalid        (:50)
 *   MF_ERR_NEEDS_PLATFORM_SETUP -> tensor.ErrNeedsPlatformSetup  (:64)
 *   MF_ERR_ALLOCATOR_EXHAUSTED  -> tensor.ErrAllocatorExhausted  (:71)
 * The remaining codes have no sentinel and surface as wrapped errors.
 * ------------------------------------------------------------------- */
enum mf_status {
    MF_OK = 0,
    MF_ERR_INVALID_ARGUMENT = -1,
    MF_ERR_DTYPE_MISMATCH = -2,
    MF_ERR_DTYPE_UNSUPPORTED = -3,
    MF_ERR_LAYOUT_UNSUPPORTED = -4,
    MF_ERR_SHAPE_MISMATCH = -5,
    MF_ERR_BACKEND_CLOSED = -6,
    MF_ERR_SHAPE_INVALID = -7,
    MF_ERR_NEEDS_PLATFORM_SETUP = -8,
    MF_ERR_ALLOCATOR_EXHAUSTED = -9,
    MF_ERR_CUDA = -10,        /* a CUDA runtime call failed */
    MF_ERR_NCCL = -11,        /* an NCCL call failed */
    MF_ERR_DEVICE_STICKY = -12 /* a kernel recorded an error in device memory */
};

/* FP8 encoder semantics. REFERENCE reproduces dtype/fp8.go:77-136 and
 * :190-249 exactly (including the subnormal shift, the exponent-15
 * saturation of E4M3 and NaN -> 0x7f). OCP is the OCP FP8 rule with
 * saturation to the largest finite value (the sm_100 cvt .satfinite
 * result) and NaN -> 0x7f. */
enum mf_compat { MF_COMPAT_REFERENCE = 0, MF_COMPAT_OCP = 1 };

typedef void* mf_stream; /* cudaStream_t */
typedef void* mf_event;  /* cudaEvent_t */
typedef struct mf_fused_kernel_s* mf_fused_kernel;
typedef struct mf_comm_s* mf_comm;
typedef struct mf_ckpt_plan_s* mf_ckpt_plan;
typedef struct mf_paged_attn_s* mf_paged_attn;
typedef struct mf_beam_select_s* mf_beam_select;
typedef struct mf_page_book_s* mf_page_book;
typedef struct mf_prefix_attn_s* mf_prefix_attn;

/* ---------------------------------------------------------------------
 * Lifecycle and errors
 * ------------------------------------------------------------------- */
int mf_abi_version(void);
/* Number of CUDA devices; works without any device (returns 0). */
int mf_device_count(int* count);
/* Select and initialise `device` for all later calls of this process.
 * Replaces the device half of tensor.Backend construction
 * (tensor/backend.go:18-68). Idempotent. */
int mf_init(int device);
/* Release library-owned device resources. After it, kernels return
 * MF_ERR_BACKEND_CLOSED until mf_init is called again
 * (tensor.Backend.Close, tensor/backend.go:65-67). */
int mf_shutdown(void);
/* Message of the last failure on this OS thread ("" if none). The pointer
 * stays valid until the next failing call on the same thread. */
const char* mf_last_error(void);
/* Copy the last error message into buf (always NUL terminated). */
int mf_last_error_copy(char* buf, size_t n);
/* Read and clear the sticky device status (MF_OK or MF_ERR_DEVICE_STICKY
 * with a code in *device_code). Synchronises the device. Backs
 * tensor.Tensor.Sync (tensor/tensor.go:53-130). */
int mf_device_status(int* device_code);
/* Device status code of a bounded wait that gave up (a bulk-copy stage that
 * never landed, or mf_wait_flag's flag that was never set). */
#define MF_DEVICE_TIMEOUT 0x7100
/* Device status code of a page number or slot outside its cache: nothing was
 * read or written there (the token counts as masked). */
#define MF_DEVICE_BAD_PAGE 0x7200
/* Device status code of a call whose device-side lengths ask for more than it
 * can index: nothing was computed. */
#define MF_DEVICE_TOO_LARGE 0x7300
/* Make `stream` wait until the int at device address `flag` equals `expect`
 * (acquire load, polled with a short sleep), for at most `max_polls` polls;
 * if it never does, record MF_DEVICE_TIMEOUT in the sticky status and let the
 * stream continue. The building block for a handshake with a peer rank or the
 * host that must not hang the GPU. No counterpart in the reference. */
int mf_wait_flag(const int* flag, int expect, int64_t max_polls, mf_stream stream);
/* Device properties used to size launches. */
int mf_device_info(int* sm_count, int* cc_major, int* cc_minor, size_t* total_bytes);

/* ---------------------------------------------------------------------
 * Memory, transfers, streams, events.  These back tensor.Backend.Upload /
 * UploadAsync / Download (tensor/backend.go:38-63) and the workspace
 * arena of runtime.WorkspaceAttacher.AttachWorkspace
 * (runtime/executor.go:42-48, sized by ir.WorkspaceLayout.Size,
 * ir/workspace.go:12-33).
 * ------------------------------------------------------------------- */
int mf_alloc(void** dptr, size_t bytes);           /* 256-byte aligned */
int mf_free(void* dptr);
int mf_host_alloc(void** hptr, size_t bytes);      /* page-locked host memory */
int mf_host_free(void* hptr);
int mf_memcpy_h2d_async(void* dst, const void* src, size_t bytes, mf_stream stream);
int mf_memcpy_d2h_async(void* dst, const void* src, size_t bytes, mf_stream stream);
int mf_memcpy_d2d_async(void* dst, const void* src, size_t bytes, mf_stream stream);
int mf_memset_async(void* dst, int value, size_t bytes, mf_stream stream);
/* Streams and events: ir.Node.StreamID and ir.SyncEvent
 * (ir/sync_event.go:14-26, ir/stream_scheduler.go:56-141) map onto these:
 * SyncEvent{Wait:false} -> mf_event_record, {Wait:true} -> mf_stream_wait_event. */
int mf_stream_create(mf_stream* stream);
int mf_stream_destroy(mf_stream stream);
int mf_stream_sync(mf_stream stream);
int mf_event_create(mf_event* event, int enable_timing);
int mf_event_destroy(mf_event event);
int mf_event_record(mf_event event, mf_stream stream);
int mf_stream_wait_event(mf_stream stream, mf_event event);
int mf_event_sync(mf_event event);
int mf_event_elapsed_ms(mf_event start, mf_event stop, float* ms);
int mf_device_sync(void);

/* ---------------------------------------------------------------------
 * K1-K3: dtype conversion.
 * Replaces the element loops of convert.BytesToFloat32 / BytesToBFloat16 /
 * BytesToFloat16 / BytesToFloat8E4M3 / BytesToFloat8E5M2
 * (dtype/convert/convert.go:85-228) and the store encoders
 * float32VectorBytes (runtime/axpy.go:171-194) and Float32AsDTypeBytes
 * (runtime/session.go:431-452).  Every conversion decodes src to float32
 * exactly as BytesToFloat32 does, then encodes with the scalar encoder of
 * dst_dtype (NewBfloat16FromFloat32 bfloat16.go:41-55, Fromfloat32
 * float16.go:109-111, NewF8E4M3FromFloat32 fp8.go:77-136,
 * NewF8E5M2FromFloat32 fp8.go:190-249).
 * src dtypes: F64 F32 F16 BF16 F8E4M3 F8E5M2 I64 I32 I16 I8 I4 U64 U32 U16 U8.
 * dst dtypes: F32 F16 BF16 F8E4M3 F8E5M2.
 * n counts logical elements; for I4 the source holds (n+1)/2 bytes.
 * ------------------------------------------------------------------- */
int mf_convert(int src_dtype, int dst_dtype, const void* src, void* dst,
               int64_t n, int compat, mf_stream stream);

/* ---------------------------------------------------------------------
 * K4: packed Int4 group dequantisation (config: 4096x14336, group 128).
 *   out[r, c] = encode_out( float32(q[r, c]) * float32(scales[r, c / group]) )
 * q is row-major [rows, cols] packed two nibbles per byte, element 2i in
 * the low nibble, sign-extended (dtype/int4.go:60-78,
 * dtype/convert/decoders.go:262-289); cols must be even so rows start on
 * byte boundaries.  scales is row-major [rows, ceil(cols/group)] of
 * scale_dtype (BF16, F16 or F32).  out_dtype is BF16 (NewBfloat16FromFloat32
 * rounding), F16 or F32.  The group scale itself has no counterpart in the
 * reference, which only sign-extends nibbles.
 * ------------------------------------------------------------------- */
int mf_int4_dequant_grouped(const void* q, const void* scales, int scale_dtype,
                            void* out, int out_dtype, int64_t rows, int64_t cols,
                            int64_t group, mf_stream stream);

/* ---------------------------------------------------------------------
 * K5: y <- y + alpha * x, in place on y.
 * Replaces axpyDevice.Axpy(y, x, count, alpha, format)
 * (runtime/axpy.go:13-15, called at :84-90) and the host loops of
 * axpyOntoHost (:115-117 for F32, :145-147 + :171-194 for BF16/F16).
 * Arithmetic: float32 multiply then float32 add, two roundings, no FMA
 * (the amd64 Go build does not contract).  fused_fma = 1 selects a single
 * rounding, which is what an arm64 Go build produces.
 * dtype: F32, BF16 or F16 (BF16/F16 decode to float32, compute, re-encode).
 * ------------------------------------------------------------------- */
int mf_axpy(void* y, const void* x, int64_t n, float alpha, int dtype,
            int fused_fma, mf_stream stream);

/* K6: out[i] = src[i] (op) scalar in float32, then encoded to dst_dtype.
 * Replaces applyScalarBroadcast (runtime/executor_math.go:195-234) and
 * its store encode (writeFloat32VectorOutput, :254-292).
 * op: 0 add, 1 sub, 2 mul, 3 div (div by 0 is rejected like :222-224). */
enum mf_scalar_op { MF_SCALAR_ADD = 0, MF_SCALAR_SUB = 1, MF_SCALAR_MUL = 2, MF_SCALAR_DIV = 3 };
int mf_scalar_broadcast(const void* src, int src_dtype, void* dst, int dst_dtype,
                        int64_t n, float scalar, int op, mf_stream stream);
/* math.linspace (runtime/executor_math.go:57-108) written straight into device
 * memory as F32, BF16 or F16 (the store encode of writeLinspaceOutput):
 * v[i] = start + float32(i) * ((stop - start) / float32(intervals)), intervals =
 * count - 1 (count when endpoint is 0), v[0] = start and v[count-1] = stop when the
 * endpoint is included. count <= 0 is MF_ERR_INVALID_ARGUMENT ("count must be
 * positive"). */
int mf_linspace(float start, float stop, int64_t count, int endpoint, void* dst, int dst_dtype,
                mf_stream stream);

/* ---------------------------------------------------------------------
 * K7: fused elementwise chains (optimizer.FusionAST, optimizer/fusion_ast.go:86-113).
 * The program is the FusionAST in postfix order: op[i] is an
 * optimizer.NodeType value (optimizer/fusion_ast.go:32-65: 1 Input,
 * 2 Constant, 3 Add, 4 Sub, 5 Mul, 6 Div, 7 Max, 8 Min, 9 Neg, 10 Abs,
 * 11 Sqrt, 12 Exp, 13 Log, 14 ReLU, 15 Sigmoid, 16 Tanh, 17 Silu,
 * 18 Gelu, 19 LeakyReLU); arg[i] is the input index for Input and the
 * index into consts for Constant, unused otherwise.
 * Per element the kernel decodes every input to float32, evaluates the
 * tree with codegen/cpu.go:126-212 semantics (binary ops and
 * Neg/Abs/ReLU/LeakyReLU in float32; Sqrt/Exp/Log/Sigmoid/Tanh/Silu/Gelu
 * in float64 rounded to float32) and encodes the result to out_dtype.
 * in_bcast[j] = 0 means input j has n elements; L > 0 means input j has L
 * elements and is read at index (i mod L) (broadcast over the last
 * dimension; the reference requires full-size inputs, cpu.go:78-85).
 * Replaces CPUKernel.Run (codegen/cpu.go:59-92).
 * ------------------------------------------------------------------- */
#define MF_FUSED_MAX_NODES 64
#define MF_FUSED_MAX_INPUTS 8
#define MF_FUSED_MAX_CONSTS 32
typedef struct mf_fused_program {
    int32_t n_nodes;
    const int32_t* op;
    const int32_t* arg;
    int32_t n_consts;
    const double* consts;
    int32_t n_inputs;
    const int32_t* in_dtype;  /* F32, F16 or BF16 */
    const int64_t* in_bcast;  /* see above; NULL = all full-size */
    int32_t out_dtype;        /* F32, F16 or BF16 */
} mf_fused_program;

/* Validate a program; picks a hand-specialised kernel when the program
 * matches one (e.g. Mul(Silu(Add(Mul(x,g),b)),y)), and emits CUDA source for
 * the expression and compiles it with NVRTC for sm_100a (the CUDA
 * counterpart of the Metal target's shader emission, codegen/metal.go:79-227;
 * 0.1-0.5 s, once per distinct program in a process).  The generated code
 * has three kernels: a bulk-copy pipeline over whole tiles of the full-size
 * inputs (16-byte aligned buffers, broadcast lengths that are multiples of 8,
 * at least one tile per SM), an 8-elements-per-lane kernel for smaller aligned
 * arrays, and an element-wise one for everything else.  MF_FUSED_JIT_DUMP=dir
 * writes each generated source to dir (a debugging aid).  Without NVRTC the
 * runtime interpreter runs the program.  Needs no device. */
int mf_fused_compile(const mf_fused_program* program, mf_fused_kernel* kernel);
int mf_fused_destroy(mf_fused_kernel kernel);
/* Which device code runs the kernel: 1 a hand-specialised body (the SwiGLU
 * chain; when its generated code's bulk-copy pipeline applies to a launch --
 * aligned buffers, at least one tile per SM -- that pipeline runs instead,
 * measured faster with the same codes), 2 CUDA source generated for this
 * expression and compiled with NVRTC for sm_100a at mf_fused_compile, 0 the
 * runtime interpreter (used when NVRTC is unavailable or MF_FUSED_JIT=0;
 * mf_last_error then gives the reason). */
int mf_fused_is_specialised(mf_fused_kernel kernel, int* specialised);
/* out: n elements of out_dtype.  If d_amax is not NULL, the kernel also
 * folds max|out| (of the encoded values, NaN ignored) into *d_amax with an
 * atomic max; *d_amax must be initialised (e.g. to 0) by the caller. */
int mf_fused_launch(mf_fused_kernel kernel, const void* const* inputs, void* out,
                    int64_t n, float* d_amax, mf_stream stream);

/* ---------------------------------------------------------------------
 * K8: per-tensor amax-scaled FP8 quantisation.  No counterpart in the
 * reference (which has no amax or scale op); built from its primitives:
 *   amax      = max |v| over the tensor (NaN ignored, Go '>' semantics)
 *   scale     = fp8_max / amax in float32 (fp8_max 448 for E4M3, 57344 for E5M2);
 *               scale = 1 when amax == 0 or amax is not finite
 *   q[i]      = encode_fp8(v[i] * scale)   (float32 multiply, compat rules)
 *   scale_inv = 1 / scale in float32 (stored for dequantisation)
 * ------------------------------------------------------------------- */
/* Fold max|src| into *d_amax (atomic max; caller initialises *d_amax). */
int mf_amax(const void* src, int src_dtype, int64_t n, float* d_amax, mf_stream stream);
/* Cast with the scale derived from *d_amax; writes *d_scale_inv if not NULL. */
int mf_fp8_scaled_cast(const void* src, int src_dtype, void* dst, int fp8_dtype,
                       const float* d_amax, float* d_scale_inv, int64_t n,
                       int compat, mf_stream stream);
/* amax + cast in one call.  d_amax is a caller-provided device float used
 * as scratch (and left holding the amax). */
int mf_fp8_quantize(const void* src, int src_dtype, void* dst, int fp8_dtype,
                    float* d_amax, float* d_scale_inv, int64_t n, int compat,
                    mf_stream stream);
/* Fused chain -> pre-cast store -> amax -> scaled FP8 in two passes:
 * pass 1 runs the fused program, writes `precast` (n values of the
 * program's out_dtype) and folds amax; pass 2 casts precast to FP8. */
int mf_fused_fp8(mf_fused_kernel kernel, const void* const* inputs, void* precast,
                 void* dst, int fp8_dtype, float* d_amax, float* d_scale_inv,
                 int64_t n, int compat, mf_stream stream);

/* ---------------------------------------------------------------------
 * K9: whole-checkpoint FP8 quantisation, tensors row-split over ranks.
 * ------------------------------------------------------------------- */
/* One contiguous chunk of one tensor owned by this rank. */
typedef struct mf_chunk_desc {
    const void* src;   /* n elements of src_dtype (F32, F16 or BF16) */
    void* dst;         /* n FP8 bytes */
    int64_t n;
    int32_t tensor;    /* index into the amax / scale_inv vectors */
    int32_t src_dtype;
} mf_chunk_desc;

/* Row split: tensor t of rows[t] x cols[t] elements is cut into `world`
 * contiguous row ranges whose sizes differ by at most one row; rank r owns
 * range r.  Writes first_row[t] and n_rows[t] for `rank`.  Host only. */
int mf_ckpt_partition(const int64_t* rows, int32_t n_tensors, int32_t world,
                      int32_t rank, int64_t* first_row, int64_t* n_rows);

/* NCCL communicator for the amax exchange.  mf_comm_unique_id writes 128
 * bytes (ncclUniqueId) on rank 0; the host sends them to every rank by any
 * means (torch.distributed store, MPI, a file); each rank then calls
 * mf_comm_init with its rank. */
int mf_comm_unique_id(void* id128);
int mf_comm_init(mf_comm* comm, int32_t world, int32_t rank, const void* id128);
int mf_comm_destroy(mf_comm comm);
/* In-place max all-reduce of a float vector in device memory. */
int mf_comm_allreduce_max_f32(mf_comm comm, float* d_vec, int64_t count, mf_stream stream);

/* The two passes on their own, for callers that run the amax exchange with
 * their own collective: pass 1 folds max|chunk| into d_amax[chunk.tensor]
 * (atomic max; the caller zeroes d_amax first); pass 2 casts every chunk
 * with the scale of d_amax[chunk.tensor] and writes d_scale_inv (if not
 * NULL).  One grouped launch per 512 chunks each. */
int mf_ckpt_amax_pass(const mf_chunk_desc* chunks, int32_t n_chunks, int32_t n_tensors,
                      float* d_amax, mf_stream stream);
int mf_ckpt_cast_pass(const mf_chunk_desc* chunks, int32_t n_chunks, int32_t n_tensors,
                      const float* d_amax, float* d_scale_inv, int fp8_dtype, int compat,
                      mf_stream stream);

/* Quantise every chunk: pass 1 folds per-tensor amax of this rank's
 * chunks into d_amax[n_tensors] (zeroed by this call), then, if comm is
 * not NULL, an NCCL max all-reduce makes d_amax global, then pass 2 casts
 * every chunk with its tensor's scale and writes d_scale_inv[n_tensors].
 * Two grouped kernel launches and at most one collective; no host sync. */
int mf_ckpt_quant_fp8(const mf_chunk_desc* chunks, int32_t n_chunks, int32_t n_tensors,
                      float* d_amax, float* d_scale_inv, int fp8_dtype, int compat,
                      mf_comm comm, mf_stream stream);

/* No counterpart in the reference.  The same quantisation as
 * mf_ckpt_quant_fp8 for callers that cannot provide device memory for the
 * per-tensor amax vector -- for example a host whose device memory all
 * belongs to another allocator, such as an executor that only holds the
 * workspace arena its graph planner sized in advance, or a deployment that
 * forbids cudaMalloc after set-up.  The amax vector lives in a static device
 * array inside the library instead (at most 4096 tensors, 16 KB per GPU,
 * held until the process exits); larger n_tensors return
 * MF_ERR_ALLOCATOR_EXHAUSTED.  Nothing is allocated.  Every call on a device
 * shares that array, so calls that overlap on the GPU race; each call zeroes
 * the entries it uses.  Every call looks the array's device address up with
 * the library's device current (nothing is cached, so a context the host
 * tears down and creates again is safe); the first call on a device also
 * loads the array there, so make it before any stream capture. */
int mf_ckpt_quant_fp8_noalloc(const mf_chunk_desc* chunks, int32_t n_chunks, int32_t n_tensors,
                              float* d_scale_inv, int fp8_dtype, int compat, mf_comm comm,
                              mf_stream stream);

/* ---------------------------------------------------------------------
 * The checkpoint quantisation step in one launch.  Replaces the same Go
 * callers as mf_ckpt_quant_fp8 (the reference itself has no quantiser; the
 * per-tensor rule is the one of mf_fp8_quantize, the encoder
 * NewF8E4M3FromFloat32 dtype/fp8.go:77-136 / NewF8E5M2FromFloat32
 * :190-249).  Same codes, scale_inv and amax as mf_ckpt_quant_fp8 with the
 * same chunk table, bit for bit.
 *
 * A plan is built once per chunk table (like the workspace plan of
 * ir.PlanWorkspace, ir/planner.go:43-96): the tensors are cut into groups of
 * consecutive tensors of at most group_bytes of this rank's source (0 = 32 MB;
 * tensor_numel, the global element count of every tensor, makes every rank cut
 * the same groups; required when world > 1, NULL = this rank's counts), the chunk table and
 * group table go to device memory, and a small exchange buffer is allocated.
 * One run is one cooperative kernel: per group an amax phase, then (one group
 * later, the group's source still in L2) a cast phase, with the per-group amax
 * exchanged between the ranks inside the kernel through the ranks' exchange
 * buffers (CUDA IPC peer memory, plain stores and system-scope flags; every
 * wait bounded, a wait that runs out leaves MF_DEVICE_TIMEOUT in the sticky
 * status).  All chunks of a plan share one source dtype (F32, F16 or BF16).
 *
 * world > 1: create on every rank, pass each rank's 64-byte ipc_handle to all
 * ranks (in rank order, world * 64 bytes) to mf_ckpt_plan_connect, and make
 * sure every rank has connected before any rank runs (a barrier).  Every rank
 * must run the plan the same number of times.  A plan is not shared between
 * streams that run at once.  Destroy on every rank after every rank's last
 * run has finished (a barrier). */
int mf_ckpt_plan_create(const mf_chunk_desc* chunks, int32_t n_chunks, int32_t n_tensors,
                        const int64_t* tensor_numel, int64_t group_bytes, int32_t world, int32_t rank,
                        int fp8_dtype, int compat, mf_ckpt_plan* plan, void* ipc_handle);
int mf_ckpt_plan_connect(mf_ckpt_plan plan, const void* ipc_handles);
/* One step: d_amax[n_tensors] (may be NULL) gets the global amax,
 * d_scale_inv[n_tensors] (may be NULL) amax / fp8_max, the chunks' dst the
 * codes.  One kernel launch; no host sync. */
int mf_ckpt_plan_run(mf_ckpt_plan plan, float* d_amax, float* d_scale_inv, mf_stream stream);
/* The same step in two launches, with the exchange fused into them instead of
 * a collective between them (same codes, amax and scale_inv, bit for bit):
 *   passes & 1  the amax pass: every source byte read once, this rank's
 *               per-tensor maxima folded into the plan's scratch; when world > 1
 *               the launch's last CTA stores them into this rank's slot of
 *               every rank's exchange buffer and sets its flag there (no
 *               collective call, no memset: the scratch of a run is cleared by
 *               the run before);
 *   passes & 2  the cast pass: its CTAs start streaming their tiles at once,
 *               wait (bounded) for every rank's flag of the run, take the
 *               maximum over the slots and cast; its CTA 0 writes d_amax and
 *               d_scale_inv (either may be NULL).
 * passes = 3 runs both; 1 then 2 (the bench times them apart) is the same.  A
 * run's amax pass must be followed by its cast pass before the next run, in
 * either form (MF_ERR_INVALID_ARGUMENT otherwise).  Two launches, no host sync. */
int mf_ckpt_plan_run_passes(mf_ckpt_plan plan, int passes, float* d_amax, float* d_scale_inv, mf_stream stream);
int mf_ckpt_plan_info(mf_ckpt_plan plan, int32_t* n_groups, int32_t* grid, int64_t* elements);
int mf_ckpt_plan_destroy(mf_ckpt_plan plan);

/* ---------------------------------------------------------------------
 * K10: a decoding step over a paged key-value cache.  The reference declares
 * the state (page_table: Int32 [capacity], paged_tensor: zeroed storage,
 * runtime/session.go:160-205) and keeps its books on the host
 * (runtime/paged_plan.go:14-177); it has no device code for it, so the
 * formulas below are the definition.
 *
 * A cache is n_pages pages of page_size tokens; token `off` of page `page`
 * has, for each of kv_heads heads, head_dim contiguous elements at
 *   page * page_stride + off * token_stride + head * head_stride   (elements)
 * for the keys and again, in another buffer, for the values: both orders of
 * heads and tokens inside a page, and padded ones, are strides.  Slot s is
 * token s % page_size of page s / page_size.  Elements are F32, BF16 or F16,
 * or FP8 codes; the value of a code of head h is decode(code) * scale_inv[h]
 * (float32 per head on the device; NULL = 1), as mf_fp8_quantize's scale_inv.
 * ------------------------------------------------------------------- */
typedef struct mf_cache_layout {
    int32_t dtype;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t page_size;
    int64_t n_pages;
    int64_t page_stride; /* elements */
    int64_t token_stride;
    int64_t head_stride;
} mf_cache_layout;

/* Page tables and slots of a step's new tokens, from the requests' lengths.
 * Request r holds lens[r] tokens and gets new_tokens[r] more (negative counts
 * as 0).  With page size P, held = ceil(lens / P), need = ceil((lens + new) / P)
 * - held and before = the sum of need over the requests in front of r:
 *   a request fits when ceil((lens + new) / P) <= max_pages, (need == 0 or
 *   before + need <= pool[1]) and its last token's number and position are
 *   31-bit; one without room in its table needs no pages;
 *   table[r][held + j] = free_pages[pool[0] + before + j],  j < need, if it fits;
 *   starts[r] = sum of new in front of r, starts[n_requests] = their total;
 *   token i = starts[r] + t: positions[i] = lens[r] + t, owner[i] = r,
 *   slots[i] = table[r][positions[i] / P] * P + positions[i] % P, or -1 if r
 *   does not fit (or that entry of the table is negative);
 *   lens_after[r] = lens[r] + new[r] if it fits, else lens[r];
 *   pool_after = {pool[0] + taken, pool[1] - taken, total of new, requests
 *   that do not fit}, taken = the largest before + need that fits.
 * pool is {index of the first free page in free_pages, number of free pages};
 * free_pages holds at least pool[0] + pool[1] page numbers.  slots, positions
 * and owner have `tokens` entries: those past the total get -1, 0, -1, and
 * tokens past `tokens` have no entry (the table is complete all the same).
 * Pages are granted to a prefix of the requests: behind the first that does not
 * fit for lack of pages nobody gets one in this call, however few it needs
 * (its need stays in `before`), and what is left stays in the pool.  So put
 * requests that must go on (a token each) in front of prompts that may wait.
 * Inputs are not changed (lens_after and pool_after are other buffers than
 * lens and pool), so a step can be planned again.  One launch, of up to
 * 2^31 - 2^16 requests. */
typedef struct mf_page_config {
    int32_t page_size;
    int32_t max_pages;    /* entries of a request's table row */
    int64_t table_stride; /* int32 entries from one row to the next, >= max_pages */
} mf_page_config;
int mf_page_assign(const mf_page_config* config, const int32_t* lens, const int32_t* new_tokens,
                   int32_t n_requests, int32_t* table, const int32_t* free_pages, const int32_t* pool,
                   int64_t tokens, int64_t* slots, int32_t* positions, int32_t* owner, int32_t* starts,
                   int32_t* lens_after, int32_t* pool_after, mf_stream stream);

/* Rotary positions.  The first rot_dim elements of a head are rot_dim / 2
 * pairs (a, b): (x[i], x[i + rot_dim/2]) in the HALF layout, (x[2i], x[2i+1])
 * in the INTERLEAVED one.  With angle = position * inv_freq[i]:
 *   a' = magnitude * (a cos - b sin),  b' = magnitude * (b cos + a sin);
 * the elements past rot_dim pass through.  inverse != 0 turns by -angle, which
 * is the gradient: dx = rope(dy, inverse).  The angle is formed and reduced in
 * float64 (a float32 product loses the phase of far positions), the rest is
 * float32, rounded once to the dtype (F32, BF16 or F16).  Positions are any
 * int32.  src and dst are [tokens, heads, head_dim] with head_dim contiguous
 * and strides in elements; dst may be src with the same strides. */
enum mf_rope_layout { MF_ROPE_HALF = 0, MF_ROPE_INTERLEAVED = 1 };
typedef struct mf_rope_config {
    int32_t dtype;
    int32_t head_dim;
    int32_t rot_dim; /* even, <= head_dim, <= 1024 */
    int32_t layout;  /* mf_rope_layout */
    float magnitude;
    const float* inv_freq; /* device, rot_dim / 2 */
} mf_rope_config;
int mf_rope(const mf_rope_config* config, int inverse, const void* src, int64_t src_token_stride,
            int64_t src_head_stride, void* dst, int64_t dst_token_stride, int64_t dst_head_stride,
            const int32_t* positions, int64_t tokens, int32_t heads, mf_stream stream);
/* The frequencies, computed in float64 and rounded to float32 once (host only):
 * base^(-2i/rot_dim), then
 *   LINEAR  divided by factor;
 *   BASE    with the base times factor^(rot_dim / (rot_dim - 2));
 *   BANDS   with turns = original_length * f / 2 pi and ramp = clamp((turns -
 *           low_turns) / (high_turns - low_turns), 0, 1):
 *           (1 - ramp) * f / factor + ramp * f. */
enum mf_rope_scaling { MF_ROPE_NONE = 0, MF_ROPE_LINEAR = 1, MF_ROPE_BASE = 2, MF_ROPE_BANDS = 3 };
int mf_rope_frequencies(int32_t rot_dim, double base, int scaling, double factor, double original_length,
                        double low_turns, double high_turns, float* inv_freq);

/* A step's queries and keys rotated (as mf_rope), keys and values written to
 * their slots: q_out[t][h] = rope(q[t][h]); cache_k at slots[t] =
 * encode(rope(k[t][h])), cache_v = encode(v[t][h]).  An FP8 cache stores
 * encode(x * (1 / scale_inv[head])) with the encoder of `compat`; any other
 * cache has the inputs' dtype.  A slot of -1 (any negative) writes no key or
 * value; one past the cache neither, and records MF_DEVICE_BAD_PAGE.  Two
 * tokens of a call must not share a slot.  q_out may be q with the same
 * strides.  Strides in elements; inputs BF16, F16 or F32. */
typedef struct mf_rope_append_config {
    mf_rope_config rope;
    mf_cache_layout cache;
    int32_t q_heads;
    int32_t compat;
    const float* k_scale_inv; /* [kv_heads] on the device, or NULL */
    const float* v_scale_inv;
    int64_t q_token_stride, q_head_stride;
    int64_t k_token_stride, k_head_stride;
    int64_t v_token_stride, v_head_stride;
    int64_t out_token_stride, out_head_stride;
} mf_rope_append_config;
int mf_rope_append(const mf_rope_append_config* config, const void* q, const void* k, const void* v, void* q_out,
                   void* k_cache, void* v_cache, const int32_t* positions, const int64_t* slots, int64_t tokens,
                   mf_stream stream);

/* Attention of one new token per request over the paged cache.  Query head h
 * reads key-value head h / (q_heads / kv_heads).  Request r sees the tokens
 * n of [first, len), len = lens[r] (clamped to the table's reach) and first =
 * max(0, len - window) (window 0 = all), token n in page table[r][n / page_size]:
 *   s_n = scale * (q . k_n)            then, if softcap > 0, softcap * tanh(s_n / softcap)
 *         + slopes[h] * (n - (len - 1))
 *   out = sum_n exp(s_n) v_n / sum_n exp(s_n),  lse = log(sum_n exp(s_n))
 * A request that sees nothing gets out = 0 and lse = -inf.  A page number
 * outside the cache masks its tokens and records MF_DEVICE_BAD_PAGE; table
 * entries past the last page are not read.
 * q and out: [n_requests, q_heads, head_dim] of q_dtype (BF16 or F16) with
 * head_dim contiguous; lse (may be NULL): float32 [n_requests, q_heads].  The
 * cache's dtype is q_dtype, F8E4M3 or F8E5M2; head_dim is a multiple of 8 (of
 * 16 for FP8) up to 256; cache buffers and strides are multiples of 16 bytes.
 * Products and sums are float32.  The weights exp(s - max) enter the product
 * with the values as two 16-bit terms: for a BF16 cache off by at most 2^-16
 * of themselves, for an F16 or FP8 cache by 2^-22 of themselves or 2^-37 of
 * the request's largest weight, whichever is more.  Exponentials are good to
 * 2^-22, capped scores to 2^-20 of themselves.  Queries over an FP8 cache are held as f16, scaled by a power of two
 * to their head's largest: an element is off by 2^-25 of that at most.  An
 * infinity among the values that are seen makes its element of the result
 * infinite or NaN.
 *
 * One run covers up to 2^31 - 2^16 requests and 2^31 - 1 tiles (16 tokens of
 * one key-value head, for up to 16 query heads); lengths that ask for more
 * record MF_DEVICE_TOO_LARGE.
 * A handle holds the description and the workspace of the split (5 to 22 MB):
 * create it once, run it for every step and layer.  A handle is not shared
 * between streams that run at once.  One launch per run, no host sync; results
 * do not depend on the order in which the parts finish. */
typedef struct mf_paged_attn_config {
    mf_cache_layout cache;
    int32_t q_dtype;
    int32_t q_heads;
    int32_t max_pages;    /* entries of a request's table row */
    int32_t window;       /* 0: all tokens */
    int64_t table_stride; /* int32 entries */
    float scale;
    float softcap;            /* 0: none; finite */
    const float* slopes;      /* [q_heads] on the device, or NULL */
    const float* k_scale_inv; /* [kv_heads] on the device, or NULL */
    const float* v_scale_inv;
    int64_t q_token_stride, q_head_stride;
    int64_t out_token_stride, out_head_stride;
} mf_paged_attn_config;
int mf_paged_attn_create(const mf_paged_attn_config* config, mf_paged_attn* handle);
int mf_paged_attn_run(mf_paged_attn handle, const void* q, const void* k_cache, const void* v_cache,
                      const int32_t* table, const int32_t* lens, int32_t n_requests, void* out, float* lse,
                      mf_stream stream);
/* Waits for the device, then frees the workspace; after mf_shutdown, too. */
int mf_paged_attn_destroy(mf_paged_attn handle);

/* ---------------------------------------------------------------------
 * K11: several continuations of a text over the paged cache of K10 (beam
 * search, or many samples of a prompt): choosing them, sharing their pages,
 * attending what they share once.  No counterpart in the reference; the
 * formulas below are the definition.
 * ------------------------------------------------------------------- */

/* The best continuations over beams and vocabulary.  Row k = entry * beams +
 * beam has vocab logits x at logits + k * row_stride (elements; F32, BF16 or
 * F16, any alignment of the dtype) and the score scores[k] so far:
 *   s(k, t) = scores[k] + x[t] - log(sum_t exp(x[t])),
 * but where ended[k] != 0 only t = end_token continues, with scores[k] as it
 * is and the logits not read.  Of each batch entry the n_out largest, in order
 * (of equal ones the lowest beam * vocab + t first):
 *   scores_after = s, tokens = t, parents = k (a row of this call: what
 *   mf_page_book_fork takes), ended_after = (t == end_token).
 * A logit of -inf is no candidate, nor is any of a row whose score or sum is
 * not finite (-inf: a beam not in use; NaN or +inf among the logits).  Where
 * there are fewer than n_out candidates, the rest is -inf, -1, -1, 0.
 * Scores are ranked in float64 and rounded once.  A term of a sum is a product of
 * up to three float32 exponentials, each good to 2^-22 of itself and 2^-23 more for
 * every octave between their arguments (a term of the size of the largest has one);
 * up to 32 terms are added in float32 (2^-21 of their sum), the rest in float64.
 * Beams whose scores are nearer to one another than that may change places.
 * beams is at most 1024, n_out at most 128, vocab at most 2^30, beams * vocab
 * below 2^31.  A handle
 * holds the workspace for batches of up to max_batch; it is not shared between
 * streams that run at once.  One launch. */
typedef struct mf_beam_select_config {
    int32_t dtype;
    int32_t vocab;
    int32_t beams;
    int32_t n_out;
    int32_t max_batch;
    int32_t end_token; /* -1: none */
    int64_t row_stride;
} mf_beam_select_config;
int mf_beam_select_create(const mf_beam_select_config* config, mf_beam_select* handle);
/* ended and ended_after may be NULL. */
int mf_beam_select_run(mf_beam_select handle, const void* logits, const float* scores, const int32_t* ended,
                       int32_t batch, float* scores_after, int32_t* tokens, int32_t* parents, int32_t* ended_after,
                       mf_stream stream);
/* The destroy calls of K11 wait for the device, then free the workspace; after mf_shutdown, too. */
int mf_beam_select_destroy(mf_beam_select handle);

/* Page tables of which rows share pages.  Beside lens, table and the pool of
 * mf_page_assign a cache then has shares[n_pages]: how many rows hold a page
 * beyond the first.  It is 0 for a page that one row holds, so that what
 * mf_page_assign grants needs no entry, and 0 for a free page; a row's page
 * that is not full belongs to it alone (fork sees to that).  A row holds
 * ceil(lens / page_size) entries of its table, at most max_pages (lens counts as
 * no more than those hold, negative as 0).  Outputs are other buffers than the
 * inputs, which stay as they are; free_pages and free_after have n_pages
 * entries, pool and pool_after are as mf_page_assign's.  What is not named below
 * is not written.
 *
 * fork: row r of n_after continues row p = parents[r] of n_before; any other p
 * (negative, or past the rows) begins empty: lens_after = 0.
 *   The first row to continue p has p's pages; every further one shares the full
 *   ones and, if the last is partly filled, gets a page of its own in its place
 *   and a move {p's page, its own, lens % page_size, 0} in moves (n_after
 *   entries, in the order of the rows).
 *   shares_after[x] = shares[x] + the further rows that share x - the rows that
 *   hold x and are not continued.  A page that this leaves without a row is
 *   free, with shares_after 0.
 *   The list of free pages becomes those, lowest number first, then
 *   free_pages[pool[0] ...]; new pages are taken from its front in the order of
 *   the rows, what is left is free_after from entry 0 on.  Where it ends too
 *   early the later rows that need a page begin empty and share nothing.
 *   table_after[r] has -1 behind the row's pages, lens_after = lens of p.
 *   pool_after = {0, pages left, moves, rows that got no page}.
 * To end rows, leave them out (or give parents of -1) and let the others go on.
 *
 * compact: a page is in use if the pool does not list it.  With limit = max(limit,
 * pages in use), the pages in use from `limit` on move, in ascending order, to the
 * lowest free ones: numbers[x] is where page x is afterwards (x itself if it
 * stays or is free), moves (n_pages / 2 entries, at least 1) has {x, numbers[x],
 * page_size, 0} of those that move, table_after the renamed table (-1 behind a
 * row's pages), shares_after the moved shares, free_after the free pages, lowest
 * first, pool_after = {0, free pages, moves, 0}.  limit 0: the pages in use
 * become 0, 1, 2, ... without a gap.  The tables name every page in use, or
 * their other holders rename theirs by `numbers`.
 * After either call run mf_page_copy on the moves before the caches are used.
 *
 * A page number outside the cache stays as it is and holds nothing.  It records
 * MF_DEVICE_BAD_PAGE where a call would change who holds the page or hand it out: in
 * fork in the tables of rows that nobody continues and of further rows, and among the
 * free pages that are taken (the pages of a row's first child are carried over as they
 * are, without a look), in compact in every row and in the whole list.  So does a list
 * of free pages past its buffer or, in compact, with a page twice; such a list counts
 * as no more pages than there are.
 * The handle holds the workspace for up to max_requests rows; it is not shared
 * between streams that run at once.  One launch. */
typedef struct mf_page_move {
    int32_t src, dst; /* pages */
    int32_t tokens;   /* the first so many */
    int32_t reserved;
} mf_page_move;
typedef struct mf_page_book_config {
    int32_t page_size;
    int32_t max_pages;    /* entries of a row of the table */
    int64_t table_stride; /* int32 entries from one row to the next, >= max_pages */
    int32_t n_pages;
    int32_t max_requests;
} mf_page_book_config;
int mf_page_book_create(const mf_page_book_config* config, mf_page_book* handle);
int mf_page_book_fork(mf_page_book handle, const int32_t* table, const int32_t* lens, int32_t n_before,
                      const int32_t* parents, int32_t n_after, const int32_t* shares, const int32_t* free_pages,
                      const int32_t* pool, int32_t* table_after, int32_t* lens_after, int32_t* shares_after,
                      int32_t* free_after, int32_t* pool_after, mf_page_move* moves, mf_stream stream);
int mf_page_book_compact(mf_page_book handle, const int32_t* table, const int32_t* lens, int32_t n_requests,
                         const int32_t* shares, const int32_t* free_pages, const int32_t* pool, int32_t limit,
                         int32_t* table_after, int32_t* shares_after, int32_t* free_after, int32_t* pool_after,
                         int32_t* numbers, mf_page_move* moves, mf_stream stream);
int mf_page_book_destroy(mf_page_book handle);

/* The first moves[i].tokens tokens of page src copied to page dst, all heads, in
 * each of n_caches caches of one layout (keys and values of every layer; a host
 * array of device addresses), for the first min(n_moves, *count) moves (count: on
 * the device, e.g. pool_after + 2; NULL: n_moves).  No page may be the dst of
 * two moves, or the src of one and the dst of another.  tokens counts as
 * 0 to page_size.  A move that names a page outside the cache is left out and records
 * MF_DEVICE_BAD_PAGE.  Elements of any dtype of a whole number of bytes; any
 * strides from 0 to 2^40, head_dim contiguous, a page's tokens below 2 GB.  One launch
 * for every 128 caches. */
int mf_page_copy(const mf_cache_layout* layout, void* const* caches, int32_t n_caches, const mf_page_move* moves,
                 int32_t n_moves, const int32_t* count, mf_stream stream);

/* mf_paged_attn_run for groups of requests that share their first tokens.
 * Requests starts[g] .. starts[g + 1] - 1 (starts: n_groups + 1 ascending
 * entries on the device) form group g and have the same pages for their first
 * shared[g] tokens, which are read once for all of them, as products on the tensor
 * cores whose rows are the group's queries; the tokens behind them, and those of
 * groups that are too small for that to pay, are read request by request.
 * out and lse are those that mf_paged_attn_run defines, for every request, with
 * the window, cap, slopes and scales of the config; shared[g] may be any number
 * of tokens (negative: 0), and a member may be shorter than it.  Requests in no
 * group share nothing.  starts that descend or leave the requests, and groups of
 * more than 2^31 - 1 tiles of tokens together, record MF_DEVICE_TOO_LARGE: nothing
 * counts as shared then, and the results are the same.
 * A request's table row names the pages of the tokens that it sees, as in
 * mf_paged_attn_run.  Shared tokens are read through the row of the first request
 * that reaches farthest into them; with a window that row names what the shorter
 * ones see, too.  What no request of the group sees is not read, and idle requests
 * may stand anywhere in it.  Where an infinity or NaN turns up among what a
 * request's rows sum, seen by it or not, all its tokens are read for it alone, so
 * that only what it sees counts.
 * Over the shared tokens, too, the weights exp(s - max) enter the product with the
 * values as two 16-bit terms, and queries over an FP8 cache are held as in
 * mf_paged_attn_run: whether a token is shared changes no bound.  head_dim,
 * dtypes, strides and alignments as there; a cache has less than 2^32 - 1 pieces
 * of the largest power of two of bytes (2^30 at most) that divides its page and token
 * strides (else MF_ERR_LAYOUT_UNSUPPORTED).
 * The workspace holds float32 parts of max_requests x q_heads x head_dim, three
 * times, and 15 to 62 MB more; it is not shared between streams that run at
 * once.  Three launches, no host sync; results do not depend on the order in
 * which parts finish. */
int mf_prefix_attn_create(const mf_paged_attn_config* config, int32_t max_requests, mf_prefix_attn* handle);
int mf_prefix_attn_run(mf_prefix_attn handle, const void* q, const void* k_cache, const void* v_cache,
                       const int32_t* table, const int32_t* lens, int32_t n_requests, const int32_t* starts,
                       const int32_t* shared, int32_t n_groups, void* out, float* lse, mf_stream stream);
/* Whether the runs that follow share whatever the groups can (1), or, as they do
 * from the start (0), where that is quicker than to read the tokens once more
 * for each request that sees them: a rule on the tokens that requests see (by their
 * lengths and the window), their numbers and the heads. */
int mf_prefix_attn_share(mf_prefix_attn handle, int32_t always);
/* How long, in nanoseconds, the runs that follow may wait for one another's parts inside a CTA: 2 * 10^9 from the start, 0
 * to 2^32 - 1 (0: not at all, every run that shares tokens is given up).  A run whose wait runs out, as where the GPU is
 * taken away from it for that long, records MF_DEVICE_TIMEOUT and comes to its end; what it wrote to out and lse counts
 * for nothing.  The runs behind it are as ever. */
int mf_prefix_attn_limit(mf_prefix_attn handle, int64_t wait_ns);
int mf_prefix_attn_destroy(mf_prefix_attn handle);

/* ---------------------------------------------------------------------
 * Measurement.  No counterpart in the reference (it has no device code).
 * mf_bw_probe moves bytes in a fixed read:write mix with the bulk-copy engine
 * alone (32 KB cp.async.bulk loads into shared memory and stores out of it,
 * no thread touches the data); its rate is the DRAM ceiling of that mix, the
 * denominator for a kernel with the same mix.  One step reads in_per_step
 * 16-byte vectors (read k of step s at src + 16 * (k * n_steps + s)) and
 * writes out_per_step (same layout in dst).  Mixes: (1,0) read-only,
 * (0,1) write-only, (1,1) copy, (1,4) decode-shaped, (2,1) cast-shaped.
 * Buffers 16-byte aligned. */
int mf_bw_probe(const void* src, int in_per_step, void* dst, int out_per_step, int64_t n_steps,
                mf_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* MFCUDA_H */
