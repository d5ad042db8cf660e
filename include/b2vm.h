/* b2vm - C ABI of the B200 device backend for VMProgram v3 bytecode.
 *
 * This is the boundary the reference's PJRT plugin (pjrt_plugin/src/plugin.cc)
 * would bind in place of its OpenCL runtime classes (pjrt_plugin/src/runtime.h).
 * Plain pointers and sizes only; no C++ or torch types cross it; nothing throws.
 * Every function that can fail returns a b2_status (0 = ok) and writes a
 * NUL-terminated message into `err` (may be NULL) of capacity `err_cap`.
 *
 * Ownership follows the reference (runtime.h:309-334): a parsed program is
 * moved into the loaded program by b2_program_load; a loaded program borrows
 * its runtime, which must outlive it; inputs are borrowed for the call; device
 * outputs returned by b2_execute_device belong to the caller and go back to the
 * runtime's size-keyed pool through b2_free.
 *
 * Threading follows the reference (runtime.h:233,301): one mutex per runtime
 * serialises Execute and host<->device copies; the pool has its own lock.
 */
#ifndef B2VM_H_
#define B2VM_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes; values are the PJRT_Error_Code values plugin.cc maps the
 * reference's bool+string errors onto (plugin.cc:634,754-761,784-790,945-972). */
typedef enum {
  B2_OK = 0,
  B2_INVALID_ARGUMENT = 3,    /* malformed blob, wrong argument count/size */
  B2_DEADLINE_EXCEEDED = 4,   /* a bounded device wait (grid barrier) ran out */
  B2_RESOURCE_EXHAUSTED = 8,  /* device allocation failed */
  B2_FAILED_PRECONDITION = 9, /* no CUDA device, lanes exceed co-residency */
  B2_UNIMPLEMENTED = 12,      /* tile op / dtype outside the backend's coverage */
  B2_INTERNAL = 13            /* CUDA runtime error */
} b2_status;

typedef struct b2_runtime b2_runtime; /* replaces pjrt_ocl::OclRuntime   (runtime.h:120-305) */
typedef struct b2_program b2_program; /* replaces pjrt_ocl::VmProgram    (runtime.h:77-104)  */
typedef struct b2_loaded b2_loaded;   /* replaces pjrt_ocl::LoadedProgram (runtime.h:309-435) */

/* What plugin.cc reads from OclRuntime::info(), ngroups(), ew_ts(), mma_t()
 * (plugin.cc:328,771-773) to describe the device and to tell the lowering
 * subprocess the tile geometry (PJRT_OCL_NLANES / PJRT_OCL_EW_TS / PJRT_OCL_MMA_T). */
typedef struct {
  char device_name[128];
  int device_ordinal;
  int sm_count;
  int cc_major, cc_minor;
  uint64_t total_mem_bytes;
  uint32_t lanes;         /* co-resident CTAs = scheduler lanes to compile for */
  uint32_t ew_ts;         /* elementwise tile size (elements) */
  uint32_t mma_t;         /* matmul output tile edge */
  uint32_t threads_per_lane;
} b2_device_info;

/* Device-side outcome of the last execute of a loaded program. */
typedef struct {
  uint32_t code;          /* 0 ok, 1 barrier wait ran out, 2 control stack overflow,
                             3 unsupported tile op reached, 4 tensor-core wait ran out,
                             5 and 6 see b2_cache_status */
  uint32_t lane;          /* lane that recorded it */
  uint32_t where;         /* barrier index / entry index */
  uint32_t detail;        /* tile op or extra information */
  uint64_t barriers;      /* grid barriers executed by lane 0 */
  uint64_t device_ns;     /* lane 0: globaltimer at exit minus at entry */
} b2_exec_status;

/* ---- runtime (OclRuntime::Create, runtime.cc:255-662) -------------------- */
b2_status b2_runtime_create(int device_ordinal, b2_runtime **out, char *err, size_t err_cap);
void b2_runtime_destroy(b2_runtime *rt);
b2_status b2_runtime_info(const b2_runtime *rt, b2_device_info *out);

/* AllocDevice / PoolAlloc / PoolFree (runtime.cc:2244-2277) and the blocking
 * WriteToDevice / ReadFromDevice (runtime.cc:2279-2301). */
b2_status b2_alloc(b2_runtime *rt, size_t bytes, void **dev_ptr, char *err, size_t err_cap);
b2_status b2_free(b2_runtime *rt, void *dev_ptr, size_t bytes);
b2_status b2_h2d(b2_runtime *rt, void *dev_dst, const void *host_src, size_t bytes, char *err, size_t err_cap);
b2_status b2_d2h(b2_runtime *rt, void *host_dst, const void *dev_src, size_t bytes, char *err, size_t err_cap);

/* ---- program (VmProgram::Parse, runtime.cc:90-251) ----------------------- */
/* Host-only: needs no CUDA device. Applies the same validation as the reference
 * parser and rejects trailing bytes like vmreader.parse (vmreader.py:314-315). */
b2_status b2_program_parse(const uint8_t *blob, size_t len, b2_program **out, char *err, size_t err_cap);
void b2_program_destroy(b2_program *prog);
uint32_t b2_program_num_inputs(const b2_program *prog);
uint32_t b2_program_num_outputs(const b2_program *prog);
uint32_t b2_program_num_lanes(const b2_program *prog);
uint32_t b2_program_num_tasks(const b2_program *prog);
uint64_t b2_program_arena_bytes(const b2_program *prog);
/* is_output: 0 = argument i, 1 = result i. dtype uses the VMProgram enum
 * (f32 0, i32 1, u32 2, bool 3, i64 4, f64 5, f16 6, bf16 7). */
uint64_t b2_program_io_bytes(const b2_program *prog, int is_output, uint32_t i);
uint32_t b2_program_io_dtype(const b2_program *prog, int is_output, uint32_t i);
uint32_t b2_program_io_rank(const b2_program *prog, int is_output, uint32_t i);
int64_t b2_program_io_dim(const b2_program *prog, int is_output, uint32_t i, uint32_t d);

/* ---- loaded program (LoadedProgram::Load, runtime.cc:735-1074) ------------ */
/* Consumes `prog` on success (it is moved into the loaded program). */
b2_status b2_program_load(b2_runtime *rt, b2_program *prog, b2_loaded **out, char *err, size_t err_cap);
void b2_loaded_destroy(b2_loaded *lp);
const b2_program *b2_loaded_program(const b2_loaded *lp);

/* LoadedProgram::Execute (runtime.cc:1103-1177): host arguments to host results,
 * synchronous; inputs[i] holds b2_program_io_bytes(prog, 0, i) bytes. */
b2_status b2_execute_host(b2_loaded *lp, const void *const *inputs, size_t n_inputs,
                          void *const *outputs, size_t n_outputs, char *err, size_t err_cap);

/* LoadedProgram::ExecuteDevice (runtime.cc:2107-2242): device arguments, device
 * results freshly taken from the pool (caller owns, returns them with b2_free);
 * synchronous like the reference's clFinish. */
b2_status b2_execute_device(b2_loaded *lp, void *const *dev_inputs, size_t n_inputs,
                            void **dev_outputs, size_t n_outputs, char *err, size_t err_cap);

/* Same, but the results are written into caller-provided device buffers and the
 * launch is enqueued on `cuda_stream` (a cudaStream_t; NULL = the runtime's own
 * stream) WITHOUT waiting for it: the asynchronous form a CUDA-stream-aware
 * caller uses to overlap copies, collectives and execution. b2_loaded_status
 * waits for that stream and reports the device status of the last launch.
 * A loaded program owns ONE arena and ONE barrier block: its launches must run
 * one after another (enqueue them on one stream, or order the streams with
 * events); two launches of the same loaded program in flight at once corrupt
 * each other. Launches may be queued back to back without fetching the status;
 * if one of them fails on the device (a wait ran out), the launches queued
 * behind it find the abort flag set, return at their first barrier without
 * writing results, and b2_loaded_status reports the first failure - so fetch
 * the status before trusting the results of a pipelined batch.
 * In/out buffers: a program buffer that is one argument and one result and that
 * the program writes (a cache updated in place; the reference copies such donated
 * buffers through its arena, runtime.cc:799-801) is updated in the RESULT's memory.
 * Pass the same address as that argument and that result and nothing is copied;
 * pass different ones and the argument is first copied into the result. */
b2_status b2_execute_device_async(b2_loaded *lp, void *const *dev_inputs, size_t n_inputs,
                                  void *const *dev_outputs, size_t n_outputs,
                                  void *cuda_stream, char *err, size_t err_cap);
b2_status b2_loaded_status(b2_loaded *lp, b2_exec_status *out, char *err, size_t err_cap);
/* The result that argument `input` shares its buffer with when that buffer is an
 * in/out buffer (see b2_execute_device_async), else -1. */
int b2_loaded_in_out_result(const b2_loaded *lp, uint32_t input);
/* Number of kernels launched by this loaded program so far. */
uint64_t b2_loaded_launch_count(const b2_loaded *lp);
/* Load-time facts about how the program was mapped to the device, for tests and
 * logs (no counterpart in the reference). `which`: 0 fused elementwise chains,
 * 1 operands forwarded in registers, 2 intermediate stores elided, 3 matmul
 * tasks, 4 matmul tasks on the tensor-core path, 5 floating-point operations of
 * all matmul tasks per execute (2 G M N K each; a task inside a loop body counts
 * once), 6 flash-attention tasks, 7 flash-attention tasks on the tensor-core path,
 * 8 strided-reduction phases whose few output tiles were re-cut by rows over all
 * lanes, 9 index of the megakernel build the program runs on (0 = the smallest;
 * the library carries several builds, each holding a subset of the tile-op
 * families, and a program runs on the smallest one that has all it uses),
 * 10 bit mask of the tile-op families the program uses, 11 full reductions
 * (RED_PART + RED_COMB) re-cut evenly over all lanes with the combine folded into
 * the same phase, 12 flash-attention tasks on the decode path (few query rows; K and
 * V rows read with 16-byte loads), 13 in/out ports, 14 phases whose units (matmuls of
 * different depth, regions, elementwise chains) were re-cut evenly over all lanes,
 * 15 groups of neighbouring row-local phases (row norms and elementwise chains over
 * the same rows) run as one pipeline per lane with the barriers between them removed,
 * 16 converts from a 16-bit dtype to f32 folded into the full sum that follows them,
 * 17 full sums taken from the row op (softmax / layer norm) that wrote their input,
 * 18 grid barriers between such a row op and its sum that were dropped (they ordered nothing any more),
 * 19 decomposed RMS norms over bf16 rows (convert, square, row sum, scalar region, two broadcast multiplies,
 * convert) run as one row op, 20 barriers dropped because the phase they closed holds nothing after that,
 * 21 whether the program runs re-planned, and of the plan: 22 fused chains and row pipelines, 23 all-pairs ops, 24 tasks of
 * the program that became part of a fused op, 25 phases.
 * Unknown `which` returns 0. */
uint64_t b2_loaded_stat(const b2_loaded *lp, int which);
/* Per-wait budget of device-side bounded waits, in nanoseconds (default 2e9). */
void b2_loaded_set_wait_budget_ns(b2_loaded *lp, uint64_t ns);
/* What the grid barrier's arrival counter (32 bits, wrapping) stands at before the next launch: results do not
 * depend on it. For tests, which reach the wrap with it. Waits for the last launch. */
b2_status b2_loaded_preset_arrivals(b2_loaded *lp, uint32_t count, char *err, size_t err_cap);
/* The time, in ns since kernel entry, at which each of the first grid barriers of
 * the last execute released (every lane had arrived, seen from lane 0) (what the reference prints under
 * PJRT_OCL_PHASE_TS, runtime.cc:2196-2240). Writes at most `cap` values and
 * returns how many were written. */
size_t b2_loaded_phase_ns(const b2_loaded *lp, uint64_t *out, size_t cap);
/* Per-lane timing, off by default (the reference's per-lane barrier timestamps,
 * VMO_TS_REC in vm_common.cl:258-282, read back and summarised by
 * runtime.cc:2196-2240). When on, every lane records its start, its exit and its
 * ARRIVAL at each of the first 64 grid barriers (globaltimer nanoseconds), which
 * is what shows straggler idle: a phase ends at its last arrival, every other
 * lane waited since its own. b2_loaded_lane_times waits for the last launch and
 * copies lanes x 66 values, lane-major: [start, exit, arrival 0 .. arrival 63];
 * returns the number of values written (0 when timing is off). */
b2_status b2_loaded_lane_timing(b2_loaded *lp, int on, char *err, size_t err_cap);
size_t b2_loaded_lane_times(b2_loaded *lp, uint64_t *out, size_t cap);

/* ---- allocation-free full sum (no counterpart in the reference) ------------ */
/* out[0] = sum of the n_elems f32 values at dev_in, for hosts that cannot
 * allocate device memory: a process whose own allocator already holds all of
 * HBM (cudaMalloc - hence b2_program_load - fails there), or a latency path that
 * cannot take the device-wide stall of cudaMalloc / cudaFree. The caller passes
 * input and output; the partial sums live in a fixed 16.3 KB array inside the
 * library (held by every GPU that loads it, until exit), which limits n_elems to
 * b2_sum_f32_static_max_elems() = 536 870 912; more is B2_INVALID_ARGUMENT.
 * Calls no cudaMalloc / cudaFree. Enqueued on `cuda_stream` (NULL = the default
 * stream) and waited for before returning. All calls on one GPU share the array:
 * calls that overlap on the GPU (other threads, other streams) race. The first
 * call on each GPU looks the array's device address up; make it before any
 * stream capture begins. Buffers 4-byte aligned (16-byte aligned input is
 * fastest). */
b2_status b2_sum_f32_static(int device_ordinal, const void *dev_in, uint64_t n_elems, void *dev_out,
                            void *cuda_stream, char *err, size_t err_cap);
uint64_t b2_sum_f32_static_max_elems(void);

/* ---- operators beside the programs (no counterpart in the reference) --------
 * What stands between a decoder block's products when the cache is shared by sequences of different lengths: rotary
 * positions with the norms of queries and keys, a paged cache, and the attention of new rows over it. They take
 * device buffers of the caller's and enqueue on `cuda_stream` (NULL = the default stream of the runtime's device)
 * without waiting; they allocate nothing and may be captured into a graph once the handles are made. The device that
 * is current when a call is made stays current; buffers are the runtime's device's.
 * A call may be made from any thread; two calls at once are independent of each other, but for what is said below
 * about b2_scratch and about rows that both write. */

/* Types of rows and pages: the VMProgram enum's values, and 8-bit floats (4 exponent, 3 mantissa bits; no infinity). */
enum { B2_F32 = 0, B2_F16 = 6, B2_BF16 = 7, B2_E4M3 = 8 };

/* rows x heads x head_dim in device memory, the last axis without gaps; strides in elements. Any alignment the type
 * has is taken; 16-byte aligned rows and heads are fastest. */
typedef struct {
  void *data;
  int64_t row_stride, head_stride;
} b2_rows;

/* Scratch for the calls that need any: partial results, and counters that every call leaves at zero. The calls that
 * share one run one after another (one stream, or streams ordered by events; graphs that hold such calls, too).
 * A loaded program's rule for its launches, for the same reason. */
typedef struct b2_scratch b2_scratch;
b2_status b2_scratch_create(b2_runtime *rt, b2_scratch **out, char *err, size_t err_cap);
void b2_scratch_destroy(b2_scratch *scratch);

/* -- rotary positions, with the norms of queries and keys in the same pass --
 * A head's row x (head_dim values) becomes, with `norm`, y = x * w / sqrt(mean(x^2) + eps), else y = x. Its first
 * rot_dim values are turned by pairs: (a, b) = (y[i], y[i + rot_dim/2]), or (y[2i], y[2i+1]) when `interleaved`,
 * by the angle position * frequencies[i]: a' = m (a cos - b sin), b' = m (a sin + b cos), m = magnitude. The rest
 * passes. In f32, the angle in 64 bits, one rounding. Sine and cosine are off by 2^-22 at most where position *
 * frequency is below 2^27, by 2^-20 at the last int32 position and a frequency of 1. */
typedef struct b2_rope b2_rope;
typedef struct {
  uint32_t head_dim, rot_dim;      /* even; head_dim <= 256, rot_dim <= head_dim, 0 = the norms alone */
  uint32_t q_heads, k_heads;       /* either may be 0: its rows are not touched then */
  uint32_t dtype;                  /* rows: B2_F32, B2_F16, B2_BF16 */
  uint32_t weight_dtype;           /* B2_F32, or `dtype` */
  uint32_t interleaved, norm;
  float eps;
  double magnitude;
  const double *frequencies;       /* host, rot_dim / 2 values, radians for each position; copied */
} b2_rope_desc;
/* Frequencies base^(-2i/rot_dim), and their forms for contexts longer than the one trained on (`factor` times):
 * LINEAR divides them by factor; STRETCH takes base * factor^(rot_dim/(rot_dim-2)); PARTS leaves those that make
 * `fast` turns or more over original_length, divides those that make `slow` or fewer, and blends between, linearly in
 * turns. (Blended over the pairs' index instead, as some checkpoints have it, the frequencies are others: hand those in.) */
enum { B2_ROPE_PLAIN = 0, B2_ROPE_LINEAR = 1, B2_ROPE_STRETCH = 2, B2_ROPE_PARTS = 3 };
b2_status b2_rope_frequencies(uint32_t rot_dim, double base, int scaling, double factor, double original_length,
                              double slow, double fast, double *out, size_t out_cap, char *err, size_t err_cap);
b2_status b2_rope_create(b2_runtime *rt, const b2_rope_desc *desc, b2_rope **out, char *err, size_t err_cap);
void b2_rope_destroy(b2_rope *rope);
/* positions: device, n_rows int32. Weights: device, head_dim values each; NULL = ones. The results may be written over
 * the inputs (same data and strides); else results and inputs lie apart, and so do the two results and the rows of each. */
b2_status b2_rope_apply(const b2_rope *rope, uint32_t n_rows, const void *positions, const b2_rows *q, const b2_rows *k,
                        const void *q_weight, const void *k_weight, const b2_rows *q_out, const b2_rows *k_out,
                        void *cuda_stream, char *err, size_t err_cap);
/* Gradients of b2_rope_apply: q and k are the inputs it had (with norm; else unused and may be NULL), dq_out and dk_out
 * the gradients of its results, dq and dk those of q and k (they may be written over dq_out and dk_out, or over q and
 * k). dq_weight / dk_weight: device, head_dim f32 each, written (not added to); either may be NULL. Sums over rows and
 * heads are in f32 in an order that does not change from call to call. `scratch` is needed for weight gradients only. */
b2_status b2_rope_apply_backward(const b2_rope *rope, b2_scratch *scratch, uint32_t n_rows, const void *positions,
                                 const b2_rows *q, const b2_rows *k, const void *q_weight, const void *k_weight,
                                 const b2_rows *dq_out, const b2_rows *dk_out, const b2_rows *dq, const b2_rows *dk,
                                 void *dq_weight, void *dk_weight, void *cuda_stream, char *err, size_t err_cap);

/* -- a paged cache of keys and values --
 * A view of pages that the caller owns: page p, slot s, head h of K starts at k_pages[p * page_stride + s *
 * slot_stride + h * head_stride] (V alike), head_dim values without a gap; base addresses and strides multiples of 16
 * bytes. e4m3 pages come with an f32 scale for each (page, slot, head): the values are code * scale. */
typedef struct b2_cache b2_cache;
typedef struct {
  uint32_t dtype;                  /* of the pages: B2_F16, B2_BF16, B2_E4M3 */
  uint32_t row_dtype;              /* of the rows that go in and out: B2_F16, B2_BF16, B2_F32; 16-bit pages: the same, or B2_F32 */
  uint32_t heads, q_heads;         /* q_heads: a multiple of heads; query head h reads cache head h / (q_heads / heads) */
  uint32_t head_dim;               /* a multiple of 16, at most 128 */
  uint32_t page_size, n_pages;     /* any page_size >= 1 */
  void *k_pages, *v_pages;
  int64_t page_stride, slot_stride, head_stride;                       /* elements */
  float *k_scales, *v_scales;                                          /* e4m3 only */
  int64_t scale_page_stride, scale_slot_stride, scale_head_stride;     /* elements */
} b2_cache_desc;
/* A batch of sequences, on the device but for its bounds. Sequence b has rows row_start[b] .. row_start[b+1] - 1 of the
 * row tensors, which are its last positions: it is `length[b]` positions long with them, and row i of its n is at
 * position length[b] - n + i (a row whose position is negative is not written to the cache, and gives zeros). Position
 * p is slot p % page_size of page pages[b * pages_stride + p / page_size]. Rows from row_start[n_seqs] on (a padded
 * batch) are left as they are. */
typedef struct {
  uint32_t n_seqs;
  uint32_t n_rows;                 /* rows that the row tensors have: at least row_start[n_seqs] */
  uint32_t max_rows;               /* the most rows a sequence of the batch has; 0 = not known */
  uint32_t max_pages;              /* entries of a sequence's page list */
  int64_t pages_stride;
  const void *row_start;           /* int32[n_seqs + 1], starting at 0 */
  const void *length;              /* int32[n_seqs] */
  const void *pages;               /* int32 */
} b2_batch;
b2_status b2_cache_create(b2_runtime *rt, const b2_cache_desc *desc, b2_cache **out, char *err, size_t err_cap);
void b2_cache_destroy(b2_cache *cache);
/* Budget of each of attention's waits on the tensor cores, in nanoseconds (default 2e9), for the calls that follow. */
void b2_cache_set_wait_budget_ns(b2_cache *cache, uint64_t ns);
/* The batch's rows of K and V into the pages. e4m3: scale = max|x| / 448 of the row, code = x / scale to the nearest
 * (ties to even); a row of zeros has scale 0; one that holds a NaN or an infinity reads back as NaN throughout.
 * Two rows of one call that name the same slot leave a mixture there. */
b2_status b2_cache_write(b2_cache *cache, const b2_batch *batch, const b2_rows *k, const b2_rows *v, void *cuda_stream,
                         char *err, size_t err_cap);
/* The batch's positions out of the pages into rows (all of a sequence: as many rows as positions). */
b2_status b2_cache_read(b2_cache *cache, const b2_batch *batch, const b2_rows *k, const b2_rows *v, void *cuda_stream,
                        char *err, size_t err_cap);
/* out = softmax(scale q k^T) v for the batch's rows over the cache, in one pass. causal: a row sees the keys up to its
 * own position, of these the last `window` (0 = all); else every position of its sequence (window must be 0). Values
 * that a row does not see never reach it, whatever they are. A row that sees nothing gives zeros. lse (may be NULL):
 * f32 [n_rows][q_heads], the logarithm of the softmax's sum (-inf for a row that sees nothing). Rows are B2_F16 or
 * B2_BF16. 0 < scale <= 1e38; max_rows x query heads to a cache head below 2^31. out must not lie over q, nor its rows
 * or heads over each other.
 * Sums, maxima and logarithms are f32. What the products take has 16 bits, each rounding off by half a step at most
 * (bf16 2^-8, f16 2^-11 of the value):
 *   single tokens (max_rows x query heads to a cache head <= 16): the weights as two values each, so that nothing is lost
 *     beside f32; bf16 rows over e4m3 pages: weight x V's scale as one f16;
 *   chunks, 16-bit pages: the weights as one value of the rows' type; e4m3 pages: f16 rows: weight x V's scale as one f16;
 *     bf16 rows: the weights as one f16, V x its scale as another.
 * e4m3 scales: each from 2^-80 to 2^103 by itself. Of the keys that a row sees together, one whose V scale is 2^19 below the
 * largest still counts in full, one 2^31 below no more, whatever its weight (f16 holds no less); chunks of bf16 rows: in full
 * down to 2^14 below the largest of its neighbours, 16 keys side by side. */
b2_status b2_cache_attend(b2_cache *cache, b2_scratch *scratch, const b2_batch *batch, const b2_rows *q, float scale,
                          int causal, uint32_t window, const b2_rows *out, void *lse, void *cuda_stream, char *err,
                          size_t err_cap);
/* Waits for the device and reports the first fault that this cache's calls met since the last report: code 5 = a page
 * number outside the cache (`lane` = sequence, `where` = entry of its list, `detail` = the number), 6 = a batch that
 * does not fit its bounds (`lane` = sequence, `detail` = the value: row_start, length or more rows than max_rows).
 * Nothing outside the buffers is touched then: such keys count as absent, such rows are left out. 4 = a wait on the
 * tensor cores ran out. Not during stream capture. */
b2_status b2_cache_status(b2_cache *cache, b2_exec_status *out, char *err, size_t err_cap);

#ifdef __cplusplus
}
#endif
#endif /* B2VM_H_ */
