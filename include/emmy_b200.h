/*
 * emmy_b200.h - C ABI of libemmyb200.so, the launch side of the B200 backend.
 *
 * What it replaces. The reference compiler writes PTX text to stdout and stops
 * there; assembling and launching happen in a remote HTTP service that is not
 * part of it (tools/run_suite.py:77-92: POST /compile {ptx} -> cubin id and
 * register counts; POST /run {entry, grid, block, smem_bytes, zero_outputs,
 * args, warmup, iters} -> median_us and outputs; the same two calls in
 * tests/test_gpu_lowering.py:70-80 and tests/test_oracle.py:236-253). This
 * library is the local stand-in for that service: it loads a module image
 * (PTX text or a cubin made by ptxas), resolves an entry point, launches it on
 * caller-owned device buffers with the geometry of meta.json, and times it
 * with CUDA events. It is a thin layer over the CUDA driver API
 * (cuModuleLoadData, cuLaunchKernelEx, cuTensorMapEncodeTiled).
 *
 * Conventions. Plain C types only. Every function returns 0 on success, a
 * CUresult value (> 0) when the driver refused, or a negative EMB_E_* code;
 * emb_last_error() then gives a text for the calling thread. The caller owns
 * all device memory (the Python host passes torch tensors' data pointers);
 * the library owns the modules it loaded until emb_module_unload. The library
 * uses the device's primary context, the one the CUDA runtime and torch use,
 * so pointers and streams are interchangeable. Calls are thread-safe as far
 * as the driver's are; there is no global state beyond the context, with one
 * exception: emb_array_sum_f32_static keeps a device array per GPU and a
 * process-wide table of its addresses, and, being written against the CUDA
 * runtime, returns cudaError_t values (> 0) where the others return CUresult
 * (so do the emb_paged_* operators).
 */
#ifndef EMMY_B200_H
#define EMMY_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define EMB_E_NO_DRIVER (-1)  /* libcuda could not be loaded (no GPU driver on this machine) */
#define EMB_E_ARGUMENT (-2)   /* an argument is out of range; see emb_last_error() */
#define EMB_E_DEVICE_STATUS (-3) /* a kernel reported a bounded wait that ran out (status word non-zero) */

/* Element types of a tensor map (values of CUtensorMapDataType are not exposed). */
enum { EMB_U8 = 0, EMB_F16 = 1, EMB_BF16 = 2, EMB_F32 = 3, EMB_U16 = 4, EMB_U32 = 5 };
/* Shared-memory swizzle of a tensor-map box. */
enum { EMB_SWIZZLE_NONE = 0, EMB_SWIZZLE_32B = 1, EMB_SWIZZLE_64B = 2, EMB_SWIZZLE_128B = 3 };

/* One kernel launch: what the runner's POST /run carries per kernel
 * (tools/run_suite.py:86-92: entry, grid, block, smem_bytes, args), with
 * `cluster_x` for modules that ask for thread-block clusters
 * (emmy_ptx/ptx.py:294-295 .reqnctapercluster). `params[i]` points at the
 * i-th kernel parameter's value: an 8-byte device pointer for a buffer
 * (the reference's only parameter kind, `.param .u64 p_<buffer>`,
 * emmy_ptx/ptx.py:288), or a 128-byte tensor map made by emb_tensor_map.
 * A module's `status` parameter is a caller-owned buffer of 8 zeroed 32-bit
 * words: [0..2] what a bounded wait that gave up recorded (code, CTA, step),
 * [4..5] work counters a persistent kernel uses and re-zeroes itself. */
typedef struct emb_launch_t {
    void* fn;
    uint32_t grid[3];
    uint32_t block[3];
    uint32_t cluster_x;  /* 0 or 1: no cluster attribute */
    uint32_t smem_bytes; /* dynamic shared memory */
    void** params;
    int32_t nparams;
    uint32_t flags; /* EMB_LAUNCH_* bits */
} emb_launch_t;

/* Programmatic dependent launch: the kernel may be scheduled while the kernel
 * before it in the stream is still running, and itself waits
 * (griddepcontrol.wait) before it touches that kernel's results. For a kernel
 * whose inputs are another kernel's `intermediate` outputs (meta.json,
 * tools/run_suite.py:81-85): hides the second launch's latency. */
#define EMB_LAUNCH_PDL 1u

/* Bind the calling thread to `device`'s primary context (retained once per
 * device). Must be called before the other functions; cheap to repeat. */
int emb_init(int device);

/* POST /compile's job after ptxas (tools/run_suite.py:77-80): make a module
 * from PTX text (NUL-terminated, JIT-compiled by the driver) or from a cubin
 * image. `nbytes` is the image size (for the record; the driver reads the
 * image's own length). */
int emb_module_load(const void* image, size_t nbytes, void** module_out);
int emb_module_unload(void* module);

/* The entry point named by meta.json's `entry` (tools/run_suite.py:88). */
int emb_get_function(void* module, const char* entry, void** fn_out);

/* Registers per thread, static shared bytes, local (spill) bytes per thread,
 * max threads per block: the `registers` figure POST /compile returns
 * (tools/run_suite.py:80,93) and its companions. Any out pointer may be NULL. */
int emb_function_info(void* fn, int* registers, int* static_smem, int* local_bytes, int* max_threads);

/* Launch one kernel / a chain of kernels in order on `stream` (a CUstream /
 * cudaStream_t; NULL is the legacy default stream). Raises the function's
 * dynamic shared memory limit when smem_bytes needs it. Asynchronous. */
int emb_launch(const emb_launch_t* launch, void* stream);
int emb_launch_chain(const emb_launch_t* launches, int n, void* stream);

/* POST /run's timing (tools/run_suite.py:91: warm-ups, then `iters` timed
 * launches; the reference reports their median): run the chain `warmup` times,
 * then `iters` times with a CUDA event pair around each run of the chain on
 * `stream`, and write the `iters` durations in microseconds to `us_out`.
 * If `flush_ptr` is non-NULL, `flush_bytes` of it are overwritten before every
 * timed run (outside the event pair) to evict the L2 cache. Synchronous. */
int emb_time_chain(const emb_launch_t* launches, int n, void* stream, int warmup, int iters,
                   void* flush_ptr, size_t flush_bytes, float* us_out);

/* The same, over `n_sets` copies of the chain bound to distinct buffers
 * (`launches` holds n_sets * chain_len descriptors, set after set): run i uses
 * set i % n_sets, so that with the sets together larger than the L2 cache
 * every timed run reads its inputs from HBM without a flush in between. One
 * event pair brackets `batch` consecutive runs (>= 1) and us_out[i] is that
 * duration divided by `batch`: with a batch of many runs the events' own cost
 * and the launch latency hidden behind the previous run drop out, which is how
 * a stream of launches behaves in production. `iters` counts batches. */
int emb_time_rotating(const emb_launch_t* launches, int chain_len, int n_sets, void* stream, int warmup, int iters,
                      int batch, float* us_out);

/* Build a tiled TMA descriptor (CUtensorMap, 128 bytes, 64-byte aligned
 * storage supplied by the caller) over a caller-owned tensor of `rank` (1..5)
 * dimensions. dims[0] is the innermost (contiguous) dimension;
 * strides_bytes[i] is the byte stride of dimension i+1 (rank-1 entries,
 * multiples of 16); box[i] is the tile extent per dimension. No counterpart
 * in the reference, whose runner protocol cannot pass a descriptor
 * (docs/DESIGN.md:860-863) and whose copy-engine path is therefore the
 * untiled cp.async.bulk (emmy_ptx/bulk.py:34-57); here the descriptor is an
 * extra kernel parameter listed in the module's launch header. */
int emb_tensor_map(void* map_out, const void* base, int dtype, int rank, const uint64_t* dims,
                   const uint64_t* strides_bytes, const uint32_t* box, int swizzle);

/* The f32 array sum (block partials, then their fold) for callers that cannot
 * allocate device memory: a plugin inside another framework's memory pool, a
 * caller in a phase where cudaMalloc's implicit synchronisation is not allowed,
 * a host with a fixed device-memory budget. It has no counterpart in the
 * reference. The compiled chain k_sum__partial -> k_sum_1_reduce needs a
 * caller-owned scratch buffer `sum__partial` of one float per block; this entry
 * point keeps that scratch in a fixed array inside the library instead
 * (EMB_STATIC_SUM_MAX_BLOCKS floats = 8 KB, resident on every GPU that loads the
 * library until the process exits) and calls no allocator of any kind.
 *   x        n floats on the current device, 16-byte aligned; n a positive multiple of 4
 *   blocks   CTAs of the first kernel = number of partials; 1..EMB_STATIC_SUM_MAX_BLOCKS,
 *            anything larger is refused with EMB_E_ARGUMENT and a text
 *   sum_out  one float on the device
 * For equal `blocks` the result is bit for bit that of the chain compiled with
 * --strict (256 threads per block, 16-byte runs, the same butterfly and tree).
 * The first call on each device looks the array's device address up
 * (cudaGetSymbolAddress, with that device current): make that first call before
 * any stream capture begins. All calls on a device share the one array, which
 * keeps the last call's partials (nothing in it has to start at zero): two calls
 * whose kernels overlap on the GPU, e.g. on different streams, race on it.
 * Asynchronous on `stream`. */
#define EMB_STATIC_SUM_MAX_BLOCKS 2048
int emb_array_sum_f32_static(const float* x, uint64_t n, uint32_t blocks, float* sum_out, void* stream);

/* ---- the exchange record of a sharded sum ------------------------------------
 * No counterpart in the reference, whose problems run on one GPU. A module whose
 * launch header lists a parameter of kind "exchange" (the last kernel of a sum)
 * takes there a DEVICE pointer to this record, or NULL for no exchange. With a
 * record the kernel stores its f32 result, with the step number in the upper half
 * of one 8-byte word, into slot [step & 1][rank] of every rank's slot memory
 * (peer stores), waits at most wait_limit_us for every rank's word of the same
 * step in its own slot memory and returns the sum of all ranks' values in rank
 * order. slot[r] is rank r's slot memory as THIS rank addresses it: 2 x
 * EMB_MAX_PEERS 8-byte words, zeroed before the first launch and mapped into
 * every rank (CUDA IPC or fabric handles; torch's symmetric memory does it). All
 * ranks must run the same number of such launches. status != 0 after a launch:
 * rank status - 1 was waited for in vain, that result and all later ones are
 * invalid, and no later launch waits again. */
#define EMB_MAX_PEERS 8
typedef struct {
    uint64_t slot[EMB_MAX_PEERS]; /* device addresses, unused entries 0 */
    uint32_t rank, world;         /* this rank, number of ranks (1..EMB_MAX_PEERS) */
    uint32_t step;                /* steps completed; start at 0, the kernels count */
    uint32_t status;              /* start at 0 */
    uint32_t wait_limit_us;       /* e.g. 2000000 */
    uint32_t reserved;            /* 0 */
} emb_peer_exchange_t;

/* ---- the serving step over a paged key-value cache -----------------------------
 * Library operators, like emb_array_sum_f32_static: run-time sizes, no IR behind
 * them, no counterpart in the reference (its attention is over whole prompts of
 * compile-time length). A step of a server calls them in this order:
 * emb_paged_assign gives the step's new tokens their places in the cache,
 * emb_paged_store normalises and rotates the new queries and keys and stores keys
 * and values there, emb_paged_attend attends one new token of each request over
 * its pages. Attention of several new tokens of a request over its pages there is
 * none: a prompt's own goes through the attention family, from dense keys that the
 * caller has normalised and rotated (emb_paged_store returns the queries only).
 *
 * Every pointer is a device address on the current device; the caller owns all of
 * them. Strides are in elements. Calls are asynchronous on `stream`, allocate
 * nothing, read nothing back and may be captured into a CUDA graph. Arguments that
 * the host can judge are refused with EMB_E_ARGUMENT and a text before anything is
 * launched; what only the device can see is stated at each call. Like
 * emb_array_sum_f32_static they return cudaError_t values (> 0) when a launch is
 * refused. */

/* The pages of a cache: element (page, token, head, d) of the keys is
 * k[page * k_stride[0] + token * k_stride[1] + head * k_stride[2] + d], of the
 * values likewise; so pages may be token-major or head-major, and keys and values
 * parts of one buffer. A SLOT is page * page_size + token. */
typedef struct {
    void* k;
    void* v;
    int64_t k_stride[3]; /* page, token, head: multiples of 16 bytes */
    int64_t v_stride[3];
    int32_t pages;     /* >= 1; pages * page_size < 2^31 */
    int32_t page_size; /* tokens in a page, >= 1, any number */
    int32_t kv_heads;
    int32_t dim;     /* 64, 128 or 256 */
    int32_t dtype;   /* EMB_F16, EMB_BF16, or EMB_U8: e4m3 codes */
    float k_scale;   /* of e4m3 codes: value = code * scale, 1.2e-38 to 3e38; else 1 */
    float v_scale;
    int32_t reserved; /* 0 */
} emb_paged_cache_t;

/* Page tables and slot maps of one step. Request b has cached[b] tokens in the
 * cache and brings fresh[b] new ones (negative counts as 0); its new tokens are
 * the step's rows starts[b] .. starts[b+1]-1. The pages they need beyond those
 * that hold cached[b] tokens come from free_pages[*free_head ..] in the order of
 * the requests and are entered into the request's row of `table`, whose other
 * entries are left as they are.
 *   slots[i], positions[i]   row i's slot and position in its request; -1 and 0 in
 *                            the rows behind the last request
 *   starts[requests + 1]     prefix sums of fresh
 *   lengths[b]               cached[b] + fresh[b]
 *   free_head_out            *free_head + pages taken
 *   report[4]                pages taken, requests refused, rows wanted beyond
 *                            `tokens`, rows wanted
 * Sums of counts stop at 2^31 - 1: starts, positions and the rows wanted are never
 * more, and rows wanted beyond `tokens` are those up to there.
 * A request is refused whole when its tokens do not fit its table row or the
 * step's `tokens` rows, or when the free pages end before its need and the need of
 * the requests before it: its slots are -1, its length stays cached[b], its table
 * row stays as it is. An entry of the table that is negative gives slot -1.
 * Outputs and `table` may share no byte with one another or with the inputs (judged
 * as for emb_paged_store). */
typedef struct {
    const int32_t* cached;
    const int32_t* fresh;
    int32_t* table;
    const int32_t* free_pages;
    const int32_t* free_head;
    int32_t* slots;
    int32_t* positions;
    int32_t* starts;
    int32_t* lengths;
    int32_t* free_head_out;
    int32_t* report;
    int64_t table_stride; /* of a request's row */
    int32_t requests;
    int32_t table_width;
    int32_t free_count; /* entries of free_pages */
    int32_t page_size;
    int32_t tokens; /* rows of slots and positions */
    int32_t reserved; /* 0 */
} emb_paged_assign_t;
int emb_paged_assign(const emb_paged_assign_t* args, void* stream);

/* Norm, rotation and store of a step's rows, in one pass:
 *   x  = q[i, h] or k[i, h];  y = x / sqrt(mean(x^2) + eps) * weight   (weight NULL: y = x)
 *   rotation of the first `rot` dims by the angles of positions[i]: rope holds, for
 *   each position, rot/2 cosines and then rot/2 sines; pair j is (y[j], y[j+rot/2]),
 *   or (y[2j], y[2j+1]) where `interleaved`:  (a c - b s, b c + a s)
 * all in f32, rounded once: q_out[i, h] in q's type, keys and values (the values as
 * they are) into slot slots[i] of the cache in the cache's type (e4m3: times
 * 1 / scale, nearest even, saturating). A slot outside the cache (negative among
 * them) stores nothing; its q_out is written. A position outside the table gives
 * NaN in the rotated dims. Two rows with the same slot leave elements of either. q_out may
 * be q, with its strides; else what is written (q_out, keys' pages, values' pages)
 * may share no byte with anything read or written (views of one buffer whose rows lie
 * between one another's are apart; memory strided in ways too odd to tell is refused).
 * A cache of 16-bit type has q's type. */
typedef struct {
    const void* q; /* [tokens, heads, dim], q_stride = row, head */
    const void* k; /* [tokens, kv_heads, dim] */
    const void* v;
    void* q_out;
    const int32_t* slots;
    const int32_t* positions; /* may be NULL where rot is 0 */
    const float* rope;        /* [rope_rows, rot] contiguous, 16-byte aligned; NULL where rot is 0 */
    const void* q_weight;     /* [dim] of q's type, or NULL */
    const void* k_weight;
    emb_paged_cache_t cache;
    int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2];
    int32_t tokens, heads;
    int32_t dtype; /* EMB_F16 or EMB_BF16 */
    int32_t rot;   /* 0, or a multiple of 16 up to dim */
    int32_t rope_rows;
    int32_t interleaved;
    float eps;
    int32_t reserved; /* 0 */
} emb_paged_store_t;
int emb_paged_store(const emb_paged_store_t* args, void* stream);

/* Attention of one token of each request over its pages:
 *   out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j,  j in [max(0, L - window), L),
 *   L = lengths[b] (negative counts as 0; window 0: all), key head h / (heads / kv_heads)
 * Key j is token j % page_size of page table[b, j / page_size]. A row without keys
 * gives 0 (lse: -inf). What pages hold behind a request's length is not looked at
 * (NaN there does no harm). A table entry outside the cache, and a length beyond
 * the table row, give NaN in the request's outputs. Scores, their maximum and sum
 * and the output are held in f32. For the product with the values a weight is off
 * by at most 2^-14 of it (bf16 caches), 2^-20 (f16 q) or 2^-11 (bf16 q over e4m3
 * codes), and over f16 and e4m3 caches by 2^-32 of the row's largest weight. Over
 * e4m3 codes an element of a bf16 q is off by up to 2^-39 of its row's largest.
 *   lse[b, h]  natural logarithm of the sum of exponentials, f32, contiguous; or NULL
 * out may be q, with its strides; else out, lse and the workspace may share no byte
 * with one another or with what is read (judged as for emb_paged_store). A cache of 16-bit type has q's type. */
typedef struct {
    const void* q; /* [requests, heads, dim], q_stride = request, head */
    void* out;
    float* lse;
    const int32_t* table;
    const int32_t* lengths;
    void* workspace; /* at least emb_paged_attend_workspace bytes, 16-byte aligned, of any content; one call at a time */
    emb_paged_cache_t cache;
    int64_t q_stride[2], out_stride[2];
    int64_t table_stride;
    int64_t workspace_bytes;
    int32_t requests, heads;
    int32_t table_width;
    int32_t dtype; /* EMB_F16 or EMB_BF16 */
    int32_t window;
    float scale;
} emb_paged_attend_t;
int emb_paged_attend(const emb_paged_attend_t* args, void* stream);
/* The bytes of workspace that a call with these sizes and types needs on the current
 * device (pointers and strides of q, out, table and the workspace are not looked
 * at); negative: an error. It does not depend on what the lengths hold. */
int64_t emb_paged_attend_workspace(const emb_paged_attend_t* args);

/* Text of the last error on the calling thread ("" if none). */
const char* emb_last_error(void);

/* ABI version of this header. */
int emb_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* EMMY_B200_H */
