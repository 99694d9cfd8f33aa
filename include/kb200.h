/*
 * kb200.h -- C ABI of the B200-native kernel library behind Kiln's GPU backend.
 *
 * The library replaces what the reference's GPU backend does with generated
 * Triton source: run the fused kernels of one optimised Kiln graph on the
 * device, writing into the single planned arena.  The host side (Python,
 * package kiln_b200) walks the Kiln graph and describes every launch with the
 * plain-old-data structs below; nothing in this interface is a torch type.
 *
 * Threading: a plan is not re-entrant (one arena), exactly like the
 * reference's GPUExecutable (kiln/gpu/runtime.py:135-136).  Launches from several
 * threads are enqueued whole, one after the other, each on its own buffers; on
 * one stream a call then sees nothing of another's.  All functions
 * return 0 on success and a negative kb200_status otherwise; the text of the
 * last failure on the calling thread is returned by kb200_last_error().
 * Nothing here aborts or throws.  Device memory is allocated, and the device
 * synchronised, only while a plan is set up: kb200_plan_create allocates the
 * plan's status word, and kb200_plan_bind allocates the library-owned scratch
 * (in BF16 mode a bf16 mirror of the arena and packed bf16 copies of constant
 * matmul operands; in the other modes copies of them laid out along K, for exact
 * FP32 the operands' tails or both operands as pairs of float16, and aligned copies of operands that a tensor map cannot
 * describe, a quarter of the free memory for all of them; a staging buffer for a fused attention whose output aliases
 * its inputs; in FP32 mode the fused attention's scratch: the operands' tails or pairs and
 * the split tiles' partial results), converts the constants (cudaDeviceSynchronize) and has a kernel look at the
 * attention mask (a blocking copy of its answer).  kb200_plan_launch and
 * kb200_kernel_launch neither allocate nor synchronise and are therefore
 * capturable into a CUDA graph; kb200_plan_status is a blocking 4-byte copy.
 */
#ifndef KB200_H
#define KB200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KB200_ABI_VERSION 7

#define KB200_MAX_RANK 6      /* iteration dims after the host collapsed contiguous ones */
#define KB200_MAX_OPERANDS 12 /* distinct tensors one fused kernel touches */
#define KB200_MAX_TAPE 96     /* scalar ops of one fused kernel */

typedef enum kb200_status {
  KB200_OK = 0,
  KB200_ERR_ARGUMENT = -1,    /* malformed descriptor, null pointer, rank/slot out of range */
  KB200_ERR_UNSUPPORTED = -2, /* well-formed but no kernel covers it (maps to NotImplementedError) */
  KB200_ERR_BOUNDS = -3,      /* an operand's span leaves the buffer it is bound to */
  KB200_ERR_CUDA = -4,        /* a CUDA call failed; message carries cudaGetErrorString */
  KB200_ERR_UNBOUND = -5,     /* launch before kb200_plan_bind */
  KB200_ERR_DEVICE_WAIT = -6, /* a bounded device-side wait ran out (see kb200_plan_status) */
  KB200_ERR_PAGES = -7        /* a cache had fewer free pages than were asked for (see kb200_cache_status; maps to MemoryError) */
} kb200_status;

/* Where a tensor lives.  Mirrors the `bases` keys of the reference's Launch
 * (kiln/gpu/codegen.py:106-116): ("arena",) ("const", name) ("input", i) ("output", i). */
typedef enum kb200_base_kind {
  KB200_BASE_ARENA = 0,
  KB200_BASE_CONST = 1,
  KB200_BASE_INPUT = 2,
  KB200_BASE_OUTPUT = 3
} kb200_base_kind;

/* Kernel classes: the four kinds the reference writes (kiln/gpu/codegen.py:532-542). */
typedef enum kb200_kclass {
  KB200_K_ELEMENTWISE = 0, /* codegen.py:284-310; also copies */
  KB200_K_ROW = 1,         /* codegen.py:312-430; LayerNorm, softmax, any row-reduction chain */
  KB200_K_REDUCE = 2,      /* codegen.py:432-482; one reduce over arbitrary dims */
  KB200_K_MATMUL = 3       /* codegen.py:484-530; batched matmul + fused epilogue */
} kb200_kclass;

/* Arithmetic mode of a matmul's operands (accumulation is always FP32).
 * FP32 corresponds to input_precision="ieee", TF32 to "tf32"
 * (codegen.py:515-516); BF16 is a backend-internal mode with no IR dtype.
 * FP32 on the tensor cores is three products of split operands -- pairs of float16 under a power of two per row where
 * the weight is frozen and suits, else pairs of TF32: within 1e-5 of exact for finite operands (the 2-norm of a row or column of results;
 * float16 pairs hold elements below 2^-84 of their row's largest to 2^-107 of that), but in the single-CTA
 * kernel on TF32 pairs NOT IEEE for non-finite ones (an infinite operand element yields NaN, see cfg[6] bit 1024 below
 * for the CUDA-core kernel that is; the others sum such rows over in float32). */
typedef enum kb200_precision {
  KB200_PREC_FP32 = 0,
  KB200_PREC_TF32 = 1,
  KB200_PREC_BF16 = 2
} kb200_precision;

/* Scalar op codes of the tape; the table follows _KernelWriter.apply
 * (codegen.py:223-248) and the prelude formulas (codegen.py:53-88). */
typedef enum kb200_opcode {
  KB200_OP_LOAD = 0,   /* a = operand slot */
  KB200_OP_IMM = 1,    /* imm = float32 literal (codegen.py:98-103) */
  KB200_OP_ACC = 2,    /* the matmul accumulator element */
  KB200_OP_ADD = 3, KB200_OP_SUB = 4, KB200_OP_MUL = 5, KB200_OP_DIV = 6,
  KB200_OP_MAX = 7, KB200_OP_MIN = 8,
  KB200_OP_NEG = 9, KB200_OP_RELU = 10, KB200_OP_EXP = 11, KB200_OP_TANH = 12,
  KB200_OP_SIGMOID = 13, KB200_OP_ERF = 14, KB200_OP_GELU_TANH = 15, KB200_OP_GELU_ERF = 16,
  KB200_OP_RSQRT = 17, KB200_OP_SQRT = 18, KB200_OP_COPY = 19,
  KB200_OP_RSUM = 20,  /* keepdim sum over the row (last iteration dim); a = value */
  KB200_OP_RMAX = 21,  /* keepdim max over the row */
  KB200_OP_STORE = 22  /* a = value, b = operand slot */
} kb200_opcode;

/* One tape entry.  Entry i defines value i; `a`/`b` name earlier entries
 * (or, for LOAD/STORE, an operand slot).  `level` is the number of row
 * reductions on the longest path from the kernel's inputs to this value
 * (the pass structure of the chunked row kernel, codegen.py:376-380). */
typedef struct kb200_tape_op {
  int32_t opcode;
  int32_t a;
  int32_t b;
  int32_t level;
  float imm;
} kb200_tape_op;

/* One tensor operand, already aligned to the kernel's iteration space:
 * stride[d] is the element stride along iteration dim d, 0 where the tensor
 * broadcasts (codegen.py:212-216 skips those dims the same way).
 * elem_offset is in float32 elements from the start of the bound buffer;
 * for the arena it already includes the planned byte offset / 4
 * (codegen.py:545-549). */
typedef struct kb200_operand {
  int32_t base_kind;   /* kb200_base_kind */
  int32_t base_index;  /* index into consts / inputs / outputs passed to kb200_plan_bind */
  int64_t elem_offset;
  int64_t stride[KB200_MAX_RANK];
} kb200_operand;

/* Iteration spaces, by class:
 *   ELEMENTWISE  iter_shape = output shape (collapsed); one launch per output.
 *   ROW          iter_shape = row dims..., inner; the reductions run over the last dim.
 *   REDUCE       iter_shape = kept dims..., reduced dims...; n_kept says where they split.
 *   MATMUL       iter_shape = batch, M, N; operands[a_slot].stride = {batch, M, K} strides,
 *                operands[b_slot].stride = {batch, K, N} strides, every other operand
 *                (epilogue inputs, outputs) is aligned to {batch, M, N}.
 */
typedef struct kb200_kernel_desc {
  int32_t kclass;      /* kb200_kclass */
  int32_t precision;   /* kb200_precision; only matmuls look at it */
  int32_t iter_rank;
  int32_t n_kept;      /* REDUCE only */
  int64_t iter_shape[KB200_MAX_RANK];
  int64_t k_extent;    /* MATMUL only: the contraction length K */
  int32_t a_slot;      /* MATMUL only */
  int32_t b_slot;      /* MATMUL only */
  int32_t n_operands;
  int32_t n_tape;
  kb200_operand operands[KB200_MAX_OPERANDS];
  kb200_tape_op tape[KB200_MAX_TAPE];
  /* Tuner configuration, opaque to the reference seam (kiln/api.py:155-162):
   * cfg[0] tile M, cfg[1] tile N, cfg[2] 128-byte K slabs per pipeline stage (1 or 2), cfg[3] pipeline stages,
   * cfg[4] split-K factor, cfg[5] implementation override (0 = library picks),
   * cfg[0] also selects the tensor-core kernel: 0 = library picks, 128 = single-CTA 128-row tiles,
   * 256 = 256-row tiles on SM pairs (cfg[1] then 128 or 256 columns, cfg[2] slabs per step).
   * cfg[6] option bits of the tensor-core matmul (0 = defaults): 512 = two MMA issuers for 64-column
   * single-CTA tiles; 1024 = an FP32-precision matmul runs on the CUDA cores instead of as three
   * products of split operands -- needed when an OPERAND may hold +-inf: the split gives inf - inf = NaN
   * tails, so the product is NaN where IEEE arithmetic gives +-inf (the Python side sets this bit on every
   * matmul when KILN_GPU_FP32_MATMUL=ieee), cfg[7] epilogue stores of the tensor-core matmul (0 = library picks,
   * 1 = ordinary global stores, never bulk tensor stores, 2 = bulk stores but always the
   * transposing lane-per-column epilogue), all 0 = library default. */
  int32_t cfg[8];
  char name[32];       /* the Kiln kernel it comes from, e.g. "k3" (diagnostics only) */
} kb200_kernel_desc;

typedef struct kb200_plan kb200_plan;

/* Library / ABI version; the host side refuses to run against a mismatch. */
int kb200_version(void);

/* Text of the last error on this thread ("" if none).  Never NULL. */
const char* kb200_last_error(void);

/* Builds a launch plan for `n` kernels on CUDA device `device`.
 * Takes the place of kiln.gpu.codegen.generate + load_module
 * (kiln/gpu/codegen.py:601-614, kiln/gpu/runtime.py:58-79): validates every
 * descriptor on the host (ranks, slots, tape references), picks the kernel
 * implementation for each class and returns KB200_ERR_UNSUPPORTED for anything
 * the reference would raise NotImplementedError on.  The descriptors are copied. */
int kb200_plan_create(const kb200_kernel_desc* descs, int n, int device, kb200_plan** out);

/* Binds device buffers.  Takes the place of the `bases` resolution in
 * GPUExecutable._run (kiln/gpu/runtime.py:164-176).  `*_bytes` are the sizes
 * of the buffers; every operand's offset + span is checked against them here,
 * on the host, before anything can run.  Buffers stay owned by the caller and
 * must outlive the launches.  May be called again to re-bind. */
int kb200_plan_bind(kb200_plan* plan, void* arena, uint64_t arena_bytes,
                    void* const* consts, const uint64_t* const_bytes, int n_consts,
                    void* const* inputs, const uint64_t* input_bytes, int n_inputs,
                    void* const* outputs, const uint64_t* output_bytes, int n_outputs);

/* Plan options, set between kb200_plan_create and kb200_plan_bind.
 * KB200_OPT_FUSE_ATTENTION (default 1): when the plan contains the reference's five-kernel
 * attention chain (K^T copy, QK^T * scale + causal mask, softmax, PV, head merge; see
 * tests/models/transformer.py:16-25 of the reference), or the seven-kernel chain of a batch of
 * sequences, run it as one fused kernel (in FP32 precision: with float32 products; on the tensor cores with the
 * operands' tails or pairs, which the projection in front writes where it can, else a small launch).  The kernel list and
 * arena offsets stay the reference's; the score buffers are then never written.  0 keeps one launch
 * per planned kernel.
 * KB200_OPT_DEPENDENT_LAUNCH (default 1): kernels are enqueued with programmatic stream
 * serialization, so that a kernel's start-up overlaps the tail of the one before it (each kernel
 * waits for its predecessor before it touches global memory).  0 = plain stream order.
 * KB200_OPT_FOLD_OPERAND_COPIES (default 1): where the plan makes a matmul's B operand N-contiguous
 * with a copy kernel (kiln/passes/buffers.py:208-217) that feeds only that matmul, the matmul reads
 * the copy's source as a K-contiguous operand and the copy is not launched.  0 launches every copy.
 * KB200_OPT_CONCURRENCY (default 1): how many plans the caller keeps in flight on this GPU at the
 * same time (a server overlapping requests on several streams).  Only a hint for the tile
 * heuristics, which the reference leaves to its autotuner (kiln/gpu/codegen.py:563-598): with n > 1 a
 * matmul counts on 1/n of the SMs and prefers fewer, wider tiles.  A matmul's results do not depend on it; with n > 1 the fused
 * attention shares no query tiles between CTAs (KB200_OPT_ATTENTION_SPLIT), which adds up in another order.
 * KB200_OPT_ABSORB_ELEMENTWISE (default 1): an elementwise kernel that directly follows a tensor-core
 * matmul and only continues it -- its one arena input is exactly the matmul's output, which nothing
 * else reads -- runs as the tail of the matmul's epilogue, and the matmul writes that kernel's output.
 * This is what the reference's plans contain behind every Linear on a [batch, tokens, d] input: its
 * fusion pass cannot take the activation or the residual add into the matmul's kernel across the
 * reshape between them (kiln/passes/fusion.py:26-35).  0 launches every planned kernel.
 * KB200_OPT_MIRROR_ONLY (default 1, BF16 and FP32 mode): a LayerNorm, matmul or fused attention whose output is read only by
 * kernels that take its bf16 mirror, or in FP32 mode its pairs of float16 (tensor-core matmul operands, the fused attention),
 * does not store the float32 values (a LayerNorm does for a row with infinities or NaN): that arena region then holds stale data, which no planned kernel reads.  0 stores
 * both, for a caller that inspects intermediate buffers.
 * KB200_OPT_FP32_ATTENTION (default 0, FP32 precision): which kernel runs the fused attention.
 * 0 = by size and by what is known of the operands: behind a projection whose results the plan can bound (frozen, behind a LayerNorm)
 * the kernel on pairs of float16, three products per float32 product, for any length above 128 tokens where it is estimated faster than the
 * CUDA-core kernel; else the kernel with three TF32 products, for sequences of whole tiles of 128 tokens whose work items fill a
 * quarter of the SMs; else, and where a matmul of the chain asked for IEEE behaviour on non-finite operands, the CUDA-core kernel.
 * 1 = always the CUDA-core kernel; 2 = always the tensor cores, on pairs of float16 where the bounds are known and else on TF32, with the pairs or
 * tails from a launch of its own (the same bits); 3 = always the tensor cores on TF32, likewise.
 * KB200_OPT_ATTENTION_SPLIT (default 1): in a launch that leaves SMs idle (one long sequence,
 * KB200_OPT_CONCURRENCY 1) the fused attention shares its long query tiles between two CTAs, which
 * merge their halves through a workspace.  0 keeps every query tile on one CTA.
 * KB200_OPT_WEIGHT_COPIES (default 1, FP32 and TF32 precision): frozen weights are also kept laid out along K
 * and, for FP32, with their tails, or as pairs of float16 beside a buffer for A's (twice the weight's own bytes in FP32, or once and three times A's bytes;
 * once in TF32), as far as a quarter of the free memory goes.  0 = every weight is read where it is, as it is beyond that.
 * KB200_OPT_FEW_TILES (default 0): asks the matmul kernel for few tiles for one of its forms instead of the one it
 * estimates to be quickest, where it covers a matmul: tile columns (64, 96 or 128) + 1000 * K splits (1, 2, 4 or 8)
 * + 10000 * (1 + how A comes, if not through a tensor map of its own: 0 a copy, 1 as float32 for BF16, 2 through four
 * maps, one per residue of its rows); a part that is 0 is left to the estimate, a form that the matmul cannot take to the other
 * kernels.
 * KB200_OPT_OTHERS_IN_FLIGHT (default 0): 1 = other plans run on this GPU at the same time, each with the whole of it
 * (KB200_OPT_CONCURRENCY 1): the last round of a matmul's tiles is then filled by them, and the tile width goes by the work
 * of all tiles instead of by rounds.  Results do not depend on it. */
typedef enum kb200_option {
  KB200_OPT_FUSE_ATTENTION = 1,
  KB200_OPT_DEPENDENT_LAUNCH = 2,
  KB200_OPT_FOLD_OPERAND_COPIES = 3,
  KB200_OPT_CONCURRENCY = 4,
  KB200_OPT_ABSORB_ELEMENTWISE = 5,
  KB200_OPT_MIRROR_ONLY = 6,
  KB200_OPT_FP32_ATTENTION = 7,
  KB200_OPT_ATTENTION_SPLIT = 8,
  KB200_OPT_WEIGHT_COPIES = 9,
  KB200_OPT_FEW_TILES = 10,
  KB200_OPT_OTHERS_IN_FLIGHT = 11
} kb200_option;
int kb200_plan_set_option(kb200_plan* plan, int option, int value);

/* Enqueues every kernel, in order, on `cuda_stream` (a cudaStream_t).
 * Takes the place of the launch loop GPUExecutable._run
 * (kiln/gpu/runtime.py:164-179).  No synchronisation, no allocation. */
int kb200_plan_launch(kb200_plan* plan, void* cuda_stream);

/* 1 when every kernel that touches a graph input or output can be pointed at another buffer without
 * binding again, so that kb200_plan_run may be used; 0 otherwise (the fused attention reads an input
 * or writes an output itself) and for an unbound plan. */
int kb200_plan_relocatable(const kb200_plan* plan);

/* kb200_plan_launch on this call's own input and output buffers (null entry: the bound one), so that
 * a call needs no copies into and out of fixed buffers.  The reference captures its launches over
 * fixed addresses and copies both ways (kiln/gpu/runtime.py:181-217).  Buffers have the size and
 * the 16-byte alignment of the bound ones, and an output overlaps no input.  Needs a relocatable
 * plan.  No synchronisation, no allocation. */
int kb200_plan_run(kb200_plan* plan, void* const* inputs, int n_inputs, void* const* outputs, int n_outputs,
                   void* cuda_stream);

/* Enqueues kernel `i` alone (profiling, autotuning).  What producers leave for it beside the arena -- bf16 mirrors, tails or float16
 * pairs of its operands -- is then as it was after their last run, whatever the arena holds. */
int kb200_kernel_launch(kb200_plan* plan, int i, void* cuda_stream);

/* Number of device kernel launches kb200_plan_launch enqueues (a Kiln kernel
 * may take more than one: packing an operand, then the matmul). */
int kb200_plan_launch_count(const kb200_plan* plan);

/* Name of the implementation chosen for kernel `i` ("ew_chain_vec4",
 * "row_layernorm", "mm_tcgen05", ...).  Never NULL for a valid i. */
const char* kb200_kernel_impl(const kb200_plan* plan, int i);

/* What runs a bound kernel `i`, in more words: for a tensor-core matmul the kernel ("mm_small", "mm_exact", "mm_pair", "mm_tc"),
 * its tile, its split and the operands it copies; for a fused attention in FP32 which of its kernels.  Valid until the thread's next call of this function. */
const char* kb200_kernel_detail(const kb200_plan* plan, int i);

/* Number of fused scalar steps kernel `i` applies per element as bound: the epilogue chain of a
 * matmul (including the steps of an elementwise or row kernel it took over, see
 * KB200_OPT_ABSORB_ELEMENTWISE), the chain of an elementwise kernel, the chain in front of a
 * register-resident row kernel's reductions; 0 for a kernel that launches nothing and for the
 * general tape kernels; -1 for a bad index or an unbound plan.  Introspection only. */
int kb200_kernel_chain_length(const kb200_plan* plan, int i);

/* Reads back the plan's device status word after the caller synchronised:
 * 0 = ok, otherwise KB200_ERR_DEVICE_WAIT with the kernel index in
 * kb200_last_error().  Device-side waits are bounded; when one runs out the
 * kernel records it here and returns normally. */
int kb200_plan_status(kb200_plan* plan);

/* Failure-path self-test (no counterpart in the reference): enqueues a one-warp kernel whose only
 * wait cannot succeed -- an mbarrier that expects two arrivals and receives one, polled a few
 * thousand times, with no copy in flight.  On expiry it records its site in the plan's status word
 * exactly as the tensor-core kernels do and returns normally; after a synchronise,
 * kb200_plan_status then returns KB200_ERR_DEVICE_WAIT (kernel 0xffff, site 0x7f) and the plan, the
 * context and the GPU stay usable.  Nothing traps, faults or spins without bound. */
int kb200_plan_selftest_wait(kb200_plan* plan, void* cuda_stream);

/* Frees the plan and any scratch it owns. */
void kb200_plan_destroy(kb200_plan* plan);

/* C = A * B on the tensor cores with operands rounded to bf16 (FP32 accumulation), for callers
 * that must not allocate.  No counterpart in the reference: it exists for hosts that cannot call
 * cudaMalloc at the point where they need a matmul -- servers that fix their device-memory
 * budget at start-up, latency-critical paths that ban allocation after initialisation, code
 * that cannot afford the device-wide synchronisation an allocation may imply.  The plan interface above obtains the packed bf16 operand
 * copies with cudaMalloc when buffers are bound; here they live in a 16 MiB array that is part
 * of the library image (every GPU that loads the library holds it until the process exits).
 *
 *   a [m, k], b [k, n], c [m, n]: row-major contiguous float32 device buffers, 16-byte aligned;
 *   n >= 64, k >= 64, both multiples of 8.
 *   Limit: 2 * (m*k + k*n) bytes (each operand rounded up to 256) must fit in 16 MiB - 256;
 *   larger shapes are refused with KB200_ERR_ARGUMENT and a message naming both numbers.
 *   status_word: optional device int, zeroed by the caller, that receives a non-zero code if a
 *   bounded device-side wait runs out; pass NULL to use (and have cleared) a word inside the array,
 *   which kb200_matmul_bf16_static_status() reads back.
 *
 * Enqueues three kernels on `cuda_stream` and returns; calls no cudaMalloc, cudaFree or any other
 * allocating routine.  The first call on a device resolves the array's device address
 * (cudaGetSymbolAddress) and raises the kernel's shared-memory limit; make that first call
 * outside any stream capture.  All calls share the one array, which keeps whatever the last call
 * left in it: nothing in it needs to start at zero except the internal status word, which each
 * call clears itself, but two calls that overlap on the GPU (different streams, or graphs
 * replayed concurrently) race on it and corrupt each other's operands. */
int kb200_matmul_bf16_static(const float* a, const float* b, float* c, int64_t m, int64_t n, int64_t k,
                             int* status_word, void* cuda_stream);

/* After the caller synchronised with the stream: 0, or KB200_ERR_DEVICE_WAIT if a bounded wait of the
 * last kb200_matmul_bf16_static call that passed status_word == NULL ran out on the current device
 * (a blocking 4-byte copy; allocates nothing).  No counterpart in the reference. */
int kb200_matmul_bf16_static_status(void);

/* ---- keys and values in pages ----------------------------------------------------------------
 * What a compiled graph cannot do: keep K and V between calls, so that the next tokens of a sequence cost their own rows
 * only.  No counterpart in the reference.  A cache holds `sequences` sequences of a model's `layers` layers in pages of
 * `page_tokens` tokens; which pages a sequence has is the same in all layers.
 *
 *   pool    [layers, 2 (K, V), pages, kv_heads, page_tokens, head_dim] of `dtype`, 16-byte aligned
 *   table   [sequences, max_pages]: the pages of a sequence in the order of its tokens, -1 behind them
 *   held    [sequences]: how many pages that is
 *   lengths [sequences]: committed tokens.  Drafted ones are written behind them (kb200_cache_append) and become
 *           committed by kb200_cache_accept.
 *   refs    [pages]: how many sequences hold the page (0 = free; a caller may keep pages for itself by counting them)
 *
 * All of it is device memory of the caller's, int32 but for the pool, consistent when the cache is created (an empty cache: table -1, the
 * rest 0; the pool may hold anything) and changed by these functions only, or by the caller between them.  Sequences may
 * share pages (kb200_cache_fork); what is written is made the writer's own first (kb200_cache_reserve).
 *
 * Every operation is enqueued on `cuda_stream`, reads its arguments and the cache's state on the device, and neither
 * allocates nor synchronises: capturable, and a replayed graph follows what the tables hold then.  Operations that change a cache use scratch
 * of its own and are ordered by the caller, like the launches of one plan; kb200_cache_attend only reads it and takes its
 * workspace from the caller, so that calls may overlap.  Page numbers and
 * indexes that are out of range are never followed: what they stand for is left out (a page of the table: read as zeros) and
 * said in the status word. */
typedef struct kb200_cache kb200_cache;

typedef enum kb200_dtype { KB200_DTYPE_FP32 = 0, KB200_DTYPE_BF16 = 1, KB200_DTYPE_FP16 = 2 } kb200_dtype;

typedef struct kb200_cache_desc {
  int32_t dtype;        /* kb200_dtype */
  int32_t layers;
  int32_t sequences;
  int32_t max_pages;    /* columns of the table; max_pages * page_tokens < 2^30 */
  int32_t pages;
  int32_t kv_heads;
  int32_t page_tokens;  /* 8, 16, 32, 64, 128 or 256 */
  int32_t head_dim;     /* a multiple of 16 up to 256 */
  void* pool;
  uint64_t pool_bytes;
  int32_t* table;
  int32_t* held;
  int32_t* lengths;
  int32_t* refs;
} kb200_cache_desc;

/* Rows of new tokens, [batch, tokens, heads, head_dim] with head_dim contiguous; strides in elements, each a multiple of 16
 * bytes like the address. */
typedef struct kb200_rows {
  void* data;
  int32_t dtype;        /* the cache's, or KB200_DTYPE_FP32: rounded to it */
  int32_t heads;
  int64_t stride[3];
} kb200_rows;

/* Bits of a cache's status word, by which kb200_cache_status tells what was left out. */
typedef enum kb200_cache_fault {
  KB200_CACHE_NO_PAGES = 1,   /* kb200_cache_reserve: fewer free pages than needed; nothing was reserved */
  KB200_CACHE_TOO_LONG = 2,   /* ... a sequence would need more than max_pages; nothing was reserved */
  KB200_CACHE_BAD_INDEX = 4,  /* a sequence, count, kept token or page out of range, a sequence given twice to kb200_cache_append,
                                 kb200_cache_weigh or kb200_cache_verify, a temperature that is negative or not finite */
  KB200_CACHE_NO_ROOM = 8,    /* a token's position has no page (see kb200_cache_reserve) */
  KB200_CACHE_SHARED = 16,    /* a write into a page that another sequence holds as well */
  KB200_CACHE_BAD_VALUE = 32  /* kb200_cache_verify: logits of an accepted token that are no distribution (NaN, +inf, all -inf) */
} kb200_cache_fault;

/* Whether kb200_cache_create takes the description; needs no GPU. */
int kb200_cache_check(const kb200_cache_desc* desc);

/* Checks the description, allocates the cache's scratch and status word on `device`.  The tables are not touched. */
int kb200_cache_create(const kb200_cache_desc* desc, int device, kb200_cache** out);

/* For every sequence s at once: it becomes what sequence sources[s] was before the call, sharing its pages; -1 leaves it
 * empty, s as it is.  Pages that nobody holds any more are free.  sources: [sequences]. */
int kb200_cache_fork(kb200_cache* cache, const int32_t* sources, void* cuda_stream);

/* Room for counts[s] tokens behind every sequence's committed ones, in pages of its own: pages that it lacks, and shared ones
 * in that range, are taken from the free pages, lowest first, in the order of the sequences and of their tokens.  A shared page all of whose
 * holders write in this call stays with the lowest of them.  The committed tokens of a replaced page are copied, in all layers; what lay behind
 * them is not kept.  All or nothing: if the pages do not suffice the cache stays as it is.  counts: [sequences]. */
int kb200_cache_reserve(kb200_cache* cache, const int32_t* counts, void* cuda_stream);

/* Keeps the first lengths[s] tokens of every sequence and frees the pages behind them; a negative entry leaves the sequence
 * as it is.  lengths: [sequences]; the cache's own array gives back what was reserved and not used. */
int kb200_cache_truncate(kb200_cache* cache, const int32_t* lengths, void* cuda_stream);

/* Moves pages so that those in use come first: the used pages behind their own number fill the free ones before it, both in
 * ascending order.  Sequences see the same tokens; the pages behind are free and keep what they held.  Pages that the caller counts for itself move
 * like the others. */
int kb200_cache_compact(kb200_cache* cache, void* cuda_stream);

/* Writes K and V of new tokens of one layer: token i < counts[b] of batch row b goes to position lengths[slots[b]] + i.
 * counts NULL: all `tokens`; slots NULL: row b is sequence b.  Needs room (kb200_cache_reserve).  No sequence twice, rows of no token
 * included; 2^30 rows at most. */
int kb200_cache_append(kb200_cache* cache, int layer, const kb200_rows* k, const kb200_rows* v, int rows, int tokens,
                       const int32_t* counts, const int32_t* slots, void* cuda_stream);

/* Commits counts[s] of the tokens drafted behind each sequence: those with the ascending indexes kept[s * kept_width + i], which
 * are moved together in all layers (kept NULL: the first ones, which stay where they are), and frees the pages behind them.
 * A sequence whose entries are not ascending, or have no pages, or would move within pages that were shared before the call, stays as it is. */
int kb200_cache_accept(kb200_cache* cache, const int32_t* counts, const int32_t* kept, int kept_width, void* cuda_stream);

/* Attention of drafted tokens: out[b, i, h] = sum_j softmax_j(scale * q[b, i, h] . k[j, g]) v[j, g], g = h * kv_heads / heads, over
 * the committed tokens j of sequence slots[b] and over the drafted ones t < counts[b] behind them with
 * mask[b * mask_stride[0] + i * mask_stride[1] + t * mask_stride[2]] != 0 (bytes; mask NULL: t <= i).  Tokens that a row does not see
 * contribute nothing, whatever they hold.  A row that sees nothing, and rows i >= counts[b], are 0.  One token per sequence is ordinary decoding.
 * scale: from 1e-30 to 1e30.  rows * tokens and 16-byte chunks of a token's heads: 2^30 each at most; tokens * heads / kv_heads: below 2^24.
 * q and out: [rows, tokens, heads, head_dim]; out has the cache's type, q that or float32 (rounded to it); they may be the same tensor, or else share no memory.  Products of 16-bit types
 * are summed in float32, the weights rounded to that type in front of V; with a float32 cache all of it is float32.  Results depend on how the call is divided among
 * the SMs (the order of sums), not on what ran before or beside it.
 * workspace: kb200_cache_attend_workspace bytes, 16-byte aligned, used by this call alone until it has run. */
uint64_t kb200_cache_attend_workspace(const kb200_cache* cache, int rows, int tokens, int heads);
int kb200_cache_attend(kb200_cache* cache, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens,
                       const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                       void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* kb200_cache_attend to a sliding window and a few first tokens, with the logarithms of the rows' sums.  Token i of a batch row stands `place` behind the committed
 * ones: places[b * tokens + i], or i where places is NULL (the depth in a tree, for masks of trees).  Places are from 0 to tokens - 1; one outside counts as the nearest of
 * these, and nothing is told: a tree goes into one call, not into several by pieces.  Of the committed tokens j it sees those with
 * j < sinks or j > lengths + place - window.  Of the drafted ones it sees what `mask` shows, whatever the window is; with mask NULL those t <= i that are
 * in the window or among the first `sinks` tokens in the same way.  window: 1 or more, 0: all tokens (sinks and places then change nothing).
 * Pages of which no row sees a token may be missing from the table (kb200_cache_release).
 * lse: NULL, or [rows, tokens, heads] by strides: log sum_j exp(scale * q k[j]) over the tokens that the row sees, -inf for rows that see nothing and rows i >= counts[b]. */
uint64_t kb200_cache_attend_window_workspace(const kb200_cache* cache, int rows, int tokens, int heads, int window, int sinks);
int kb200_cache_attend_window(kb200_cache* cache, int layer, const kb200_rows* q, const kb200_rows* out, int rows, int tokens,
                              const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                              int window, int sinks, const int32_t* places, float* lse, const int64_t* lse_stride,
                              void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* Gives back the pages that a window has left: those of which every token j has j >= sinks and j <= lengths[s] - window, so that no token to come sees it (places of 0
 * and more).  Their entries become -1; held and lengths stay.  What needs them afterwards (a larger window, kb200_cache_attend, room behind a sequence that was truncated into
 * them) is told KB200_CACHE_BAD_INDEX. */
int kb200_cache_release(kb200_cache* cache, int window, int sinks, void* cuda_stream);

/* The weight that the tokens of a sequence draw: out[s, j] = weights[s, j] + sum over i < counts[b] and heads h of exp(scale * q[b, i, h] . k[j, g] - lse[b, i, h]) for the tokens
 * j that token i of batch row b (s = slots[b]) sees, as in kb200_cache_attend, whose lse makes them its weights.  Rows whose lse is -inf add nothing.  All other entries of out
 * are weights'.  committed: 0, the tokens are those drafted behind the committed ones, as in kb200_cache_attend; else they are the last counts[b] of the committed ones (what
 * kb200_cache_accept has taken, in its order).  weights and out: float32 [sequences, max_pages * page_tokens], a row `stride` elements behind the last; weights NULL: zeros; out may be weights.
 * No sequence twice.  Tokens whose page is missing (kb200_cache_release) draw nothing and are told KB200_CACHE_BAD_INDEX.  Sums are float32; every key's are taken in the same order in every call. */
int kb200_cache_weigh(kb200_cache* cache, int layer, const kb200_rows* q, const float* lse, const int64_t* lse_stride, int rows, int tokens,
                      const uint8_t* mask, const int64_t* mask_stride, const int32_t* counts, const int32_t* slots, float scale,
                      int committed, const float* weights, int64_t weights_stride, float* out, int64_t out_stride, void* cuda_stream);

/* Keeps keep[s] of every sequence's committed tokens and drops the others, in all layers: the first `sinks`, of the rest the last `recent`, and of what then lacks the heaviest
 * by weights[s] (of equal ones the first; NaN is heaviest); fewer than the first and last ones where keep[s] is less.  They keep their order and become the sequence's first keep[s]
 * tokens (whose indexes are then no positions in a text: lengths, windows and places count what is left); the pages behind them are free, what was reserved too.  A negative entry, or one of lengths[s] and more, leaves the sequence as it is.
 * out[s]: the weights of the tokens that the sequence then has, zeros behind them.  weights and out: as in kb200_cache_weigh; out may be weights.
 * A sequence whose tokens would move within pages that were shared before the call, or that would keep tokens of pages that it does not have (kb200_cache_release), stays
 * as it is.
 * workspace: kb200_cache_evict_workspace bytes, 16-byte aligned, used by this call alone until it has run. */
uint64_t kb200_cache_evict_workspace(const kb200_cache* cache);
int kb200_cache_evict(kb200_cache* cache, const float* weights, int64_t weights_stride, const int32_t* keep, int recent, int sinks,
                      float* out, int64_t out_stride, void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* Rows over a vocabulary, [batch, tokens, vocabulary] with the last contiguous; strides in elements. */
typedef struct kb200_scores {
  const void* data;
  int32_t dtype;        /* kb200_dtype */
  int32_t pad;
  int64_t stride[2];
} kb200_scores;

/* Which drafted tokens the model accepts, and the token that follows them, by given random numbers: what is returned is distributed as the model's own samples.
 *   drafted [rows, tokens]: token i < counts[b] of a batch row, as appended behind sequence slots[b].  Token 0 is not in question (it followed the last step).
 *   parents [rows, tokens] by parents_stride: the token i that each one follows, smaller than itself (NULL: a chain); -1: none, it is never asked for.
 *   logits: the model's of what follows each token.  p_i = softmax(logits[b, i] / temperature[b]); temperature 0: all of it on the largest logit (the first of equal ones);
 *     NULL: 1.
 *   draft: the probabilities by which the tokens that follow token i were drawn, each for itself; NULL (and for temperature 0): they were chosen without chance.
 *   uniform [rows, tokens]: numbers from [0, 1), one for each drafted token and, in place 0, one for the token that follows.
 * From a = 0 on, with r = p_a and R = 1, the tokens c that follow a are asked for in their order.  With x = drafted[b, c], c is accepted if
 * uniform[b, c] * draft[b, a, x] * R < r(x) (without draft: uniform[b, c] * R < r(x)); then it takes a's place.  If not, r becomes max(r / R - draft[b, a], 0) (without: r(x)
 * becomes 0) and R its sum, unless that is 0.  In the end following[s] is the first v at which r, summed up, exceeds uniform[b, 0] times its sum.
 * n_accepted [sequences], accepted [sequences, tokens] (-1 behind): as kb200_cache_accept takes them; sequences without a row, or with counts[b] 0: 0, and -1 in following.
 * Numbers are compared as if computed in float64, with probabilities that are off by 4e-12 of themselves at most (below 2^-1000 of a row's largest they are 0) and sums of what a draft leaves by
 * 1e-10.  (Where a draft leaves no more than such errors, because it is the model itself, the token that follows is one that the model may draw.)  If the logits of an accepted token are
 * no distribution the row ends there, with -1 in following.  tokens: 512 at most.
 * workspace: kb200_cache_verify_workspace bytes, 16-byte aligned, used by this call alone until it has run. */
uint64_t kb200_cache_verify_workspace(const kb200_cache* cache, int rows, int tokens, int vocab);
int kb200_cache_verify(kb200_cache* cache, const kb200_scores* logits, const kb200_scores* draft, int rows, int tokens, int vocab, const int32_t* drafted,
                       const int32_t* parents, int64_t parents_stride, const float* uniform, const float* temperature, const int32_t* counts, const int32_t* slots,
                       int32_t* n_accepted, int32_t* accepted, int32_t* following, void* workspace, uint64_t workspace_bytes, void* cuda_stream);

/* After the caller synchronised: 0, or what the operations since the last call left out (KB200_ERR_PAGES where pages
 * were short, else KB200_ERR_BOUNDS; the text names the bits).  A blocking 4-byte copy; what it tells is cleared when it
 * returns. */
int kb200_cache_status(kb200_cache* cache);

void kb200_cache_destroy(kb200_cache* cache);

#ifdef __cplusplus
}
#endif
#endif /* KB200_H */
