/*
 * thompiler runner: the C ABI that loads and launches the PTX compile.py
 * emits, on the local B200.  It replaces the hackathon's remote GPU runner,
 * whose HTTP contract is the reference's docs/API.md; each call below names
 * the part of that contract it stands in for.
 *
 * Conventions
 *   - Every call returns a thr_status; 0 is success.  Nothing is thrown or
 *     aborted across the ABI.  thr_last_error() gives the message of the
 *     calling thread's last failure (ptxas / JIT log text included).
 *   - Handles (modules, functions, streams, device pointers) are plain
 *     uint64_t; a stream of 0 is the legacy default stream.
 *   - One CUDA context per process and device: the device's primary
 *     context, shared with any other runtime in the process (PyTorch).
 */
#ifndef THOMPILER_RUNNER_H
#define THOMPILER_RUNNER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Failure stages of docs/API.md:56-60, plus two local ones. */
typedef enum {
    THR_OK = 0,
    THR_ERR_PTXAS = 1,      /* the PTX did not assemble / JIT        */
    THR_ERR_LOOKUP = 2,     /* unknown module, entry or global       */
    THR_ERR_RUN = 3,        /* the launch or a copy failed           */
    THR_ERR_REQUEST = 4,    /* bad arguments                         */
    THR_ERR_TIMEOUT = 5,    /* the work did not finish in time       */
    THR_ERR_CUDA = 6,       /* CUDA unavailable / other CUDA failure */
} thr_status;

/* Argument kinds of a /run request (docs/API.md:44-52).  Seeded inputs are
 * generated by the caller on the host; here every input is host data. */
typedef enum {
    THR_ARG_INPUT = 0,      /* copied host -> device before the launches      */
    THR_ARG_OUTPUT = 1,     /* zeroed before the launches, copied back after  */
} thr_arg_kind;

typedef struct {
    void *host;             /* host buffer: source (input) or destination (output) */
    uint64_t nbytes;
    int32_t kind;           /* thr_arg_kind */
    int32_t zero_each;      /* 1: re-zeroed before EVERY launch (meta "zero_outputs") */
} thr_arg;

/* Library ABI version (bumped on any signature change). */
int thr_version(void);

/* Make `device` current in this thread and retain its primary context. */
int thr_init(int device);

/* Device facts a launch plan needs. */
int thr_device_info(int device, int *sm_count, int *cc_major, int *cc_minor,
                    char *name, size_t name_len);

/* POST /compile (docs/API.md:12-24): JIT-assemble a PTX module for the
 * current device.  On THR_ERR_PTXAS the JIT error log is in thr_last_error.
 * `log` (may be NULL) receives the JIT info log (ptxas -v style). */
int thr_module_load(const char *ptx, uint64_t *module, char *log, size_t log_len);
int thr_module_unload(uint64_t module);

/* The "entry_points" / "registers" of the /compile answer: look up an entry
 * and read its resource use. */
int thr_get_function(uint64_t module, const char *entry, uint64_t *function);
int thr_function_attrs(uint64_t function, int *num_regs, int *max_threads,
                       int *static_smem, int *local_bytes);

/* Address and size of a module-scope .global variable (tuned kernels keep
 * scratch words and tensor maps there). */
int thr_module_global(uint64_t module, const char *name, uint64_t *dptr, uint64_t *nbytes);

/* One launch with device-pointer arguments (each args[i] is a device
 * address passed as the i-th .u64 parameter).  Raises the dynamic shared
 * memory limit of `function` when smem_bytes > 48 KiB.  Asynchronous. */
int thr_launch(uint64_t function, const uint32_t grid[3], const uint32_t block[3],
               uint32_t smem_bytes, const uint64_t *args, int nargs, uint64_t stream);

/* thr_launch with flags (no counterpart in the reference, whose remote runner launches one
 * request at a time).  THR_LAUNCH_OVERLAP_PREVIOUS: programmatic dependent launch -- the
 * kernel may start while the stream's previous kernel is finishing (after that kernel's CTAs
 * execute griddepcontrol.launch_dependents), so its launch latency and set-up overlap the
 * previous kernel's tail.  Only for kernels that execute griddepcontrol.wait before their
 * first access to global data (the tuned families whose launch record carries "pdl": true);
 * a copy or other non-kernel work before it on the stream is still waited for in full.
 * Without the driver entry point the launch is an ordinary one. */
#define THR_LAUNCH_OVERLAP_PREVIOUS 1u
int thr_launch_ex(uint64_t function, const uint32_t grid[3], const uint32_t block[3],
                  uint32_t smem_bytes, const uint64_t *args, int nargs, uint64_t stream,
                  uint32_t flags);

/* POST /run (docs/API.md:26-52) on host buffers: copy inputs in, zero the
 * outputs, run `warmup` untimed and `iters` timed launches (re-zeroing the
 * zero_each outputs before every launch), copy outputs back, and report the
 * median launch time.  Device buffers are owned by the runner and reused
 * between calls.  Waits at most timeout_s seconds for the work. */
int thr_run(uint64_t function, const uint32_t grid[3], const uint32_t block[3],
            uint32_t smem_bytes, const thr_arg *args, int nargs, int warmup, int iters,
            double timeout_s, float *median_us, uint64_t stream);

/* A tensor map a tuned kernel reads from a module global, described for
 * thr_run_ex: it is encoded for the device buffer of argument `arg`. */
typedef struct {
    const char *global;     /* module .global receiving the 128-byte map    */
    int32_t arg;            /* index (in args) of the buffer it maps        */
    int32_t dtype_code;     /* as thr_tensor_map                            */
    int32_t rank;
    int32_t swizzle;
    uint64_t dims[5];       /* innermost first                              */
    uint64_t strides[4];    /* bytes, dims 1..rank-1                        */
    uint32_t box[5];
} thr_tmap_spec;

/* thr_run for kernels whose tuned launch reads tensor maps: after staging
 * the arguments, binds the module's tensor-map set for the staged buffers
 * (thr_tmap_bind) and marks it read by each launch.  Same POST /run
 * semantics otherwise (docs/API.md:26-52). */
int thr_run_ex(uint64_t module, uint64_t function, const uint32_t grid[3], const uint32_t block[3],
               uint32_t smem_bytes, const thr_arg *args, int nargs, const thr_tmap_spec *tmaps,
               int ntmaps, const char *ptr_table, int warmup, int iters, double timeout_s,
               float *median_us, uint64_t stream);

/* One request of thr_run_batch: a POST /run with a single launch. */
typedef struct {
    uint64_t module;                /* module of `function` (for tensor maps; 0 without maps) */
    uint64_t function;
    uint32_t grid[3];
    uint32_t block[3];
    uint32_t smem_bytes;
    int32_t nargs;
    const thr_arg *args;
    const thr_tmap_spec *tmaps;
    int32_t ntmaps;
    const char *ptr_table;
} thr_run_desc;

/* Several independent POST /run requests (docs/API.md:26-52, one launch each, outputs zeroed
 * first) on host buffers, overlapped: request r's inputs cross PCIe on one stream while request
 * r-1's kernel runs on a second and earlier requests' outputs come back on a third, so both
 * copy directions are busy at once (pass pinned host memory, else the copies serialise).  No
 * request may read another's outputs.  Requests of one module are fine, tensor maps included:
 * each binds its own tensor-map set (thr_tmap_bind); past the module's number of sets, a set's
 * re-encoding waits for the earlier request that read it.  Returns once every output is back
 * in host memory, waiting at most timeout_s seconds. */
int thr_run_batch(const thr_run_desc *runs, int nruns, double timeout_s);

/* Tensor maps of a tuned launch on device pointers (no counterpart in the reference, whose
 * runner has no TMA).  A tuned module reads its maps from module globals; laid out as a ring
 * (every spec naming one global of sets x ntmaps maps of 128 bytes, and ptr_table holding sets x
 * ntmaps buffer addresses) it keeps several sets, and its kernel uses the set whose recorded
 * addresses equal its parameters -- so launches of one module on different buffers may be in
 * flight at once, on any streams.  thr_tmap_bind returns (in *set) the set encoded for the
 * buffers args[tmaps[i].arg] (args: the launch's device pointers in argument order); when no set
 * is, it re-encodes the least recently used one with stream-ordered copies on `stream`, after
 * the last launch that read that set.  Call thr_tmap_launched right after issuing the launch
 * (same stream) so a later re-encoding waits for it.  A set read by a launch captured into a
 * CUDA graph is kept for good (and a call on new buffers refused once every set is, or could be
 * mistaken for one that is); a set must be encoded, and its upload complete, before a capture
 * reads it (launch once on the same buffers and synchronise first).  Maps in separate globals
 * (one per spec) form a single set.  Threads that launch one module this way hold a lock of their
 * own from the binding to the report, or another one's binding may re-encode the set in between;
 * thr_launch_prepared, thr_run_ex and thr_run_batch hold the module's. */
int thr_tmap_bind(uint64_t module, const thr_tmap_spec *tmaps, int ntmaps, const char *ptr_table,
                  const uint64_t *args, int nargs, uint64_t stream, int *set);
int thr_tmap_launched(uint64_t module, int set, uint64_t stream);

/* Everything of a launch on device pointers that stays the same from call to call: filled in once,
 * read by each thr_launch_prepared. */
typedef struct {
    uint64_t module;                /* of `function` (for tensor maps; 0 without maps) */
    uint64_t function;
    uint32_t grid[3];
    uint32_t block[3];
    uint32_t smem_bytes;
    uint32_t flags;                 /* as thr_launch_ex */
    int32_t nargs;
    int32_t ntmaps;
    const uint32_t *align;          /* per argument: the power of two its address must be a multiple of, 0 for any
                                       (NULL: any for all) */
    const thr_tmap_spec *tmaps;
    const char *ptr_table;
} thr_launch_desc;

/* One launch of `desc` on args[nargs]: addresses checked against `align` (THR_ERR_REQUEST before
 * anything is issued), tensor maps bound, launched and their reader reported in one call. */
int thr_launch_prepared(const thr_launch_desc *desc, const uint64_t *args, uint64_t stream);

/* A 2-D..5-D tiled TMA descriptor (CUtensorMap, 128 bytes) for `base`.
 * dtype_code: 0 = f16, 1 = bf16, 2 = f32; swizzle: 0 none, 1 = 32B,
 * 2 = 64B, 3 = 128B.  dims / box innermost first; strides in bytes for
 * dims 1..rank-1. */
int thr_tensor_map(void *out128, int dtype_code, int rank, uint64_t base, const uint64_t *dims,
                   const uint64_t *strides_bytes, const uint32_t *box, int swizzle);

/* Stream-ordered host -> device copy, a blocking device -> host copy (e.g.
 * a kernel's error word), and a device-wide synchronise. */
int thr_memcpy_htod(uint64_t dst, const void *src, uint64_t nbytes, uint64_t stream);
int thr_memcpy_dtoh(void *dst, uint64_t src, uint64_t nbytes);
int thr_synchronize(void);

/* Release the runner's cached device buffers. */
int thr_release_buffers(void);

/* Copy the calling thread's last error message into buf (NUL-terminated). */
int thr_last_error(char *buf, size_t n);

/* Allocation-free f32 array sum: out[0] = sum of x[0..n).  No counterpart in
 * the reference; it exists for callers that cannot call cudaMalloc -- those
 * whose device memory belongs to their own allocator or pool, and latency-
 * critical paths where cudaMalloc / cudaFree would block or synchronise the
 * device.  The caller passes device pointers (x 16-byte aligned, out 4-byte
 * aligned); the only scratch is a static device array of
 * THR_NOALLOC_MAX_CTAS partials plus a counter (16,640 bytes) that every GPU
 * loading this library holds until exit.  ctas = 0 picks 4 CTAs per SM; more
 * than THR_NOALLOC_MAX_CTAS is rejected with THR_ERR_REQUEST.  The first call
 * on a device, and the first after a cudaDeviceReset, looks up the array's
 * address (make those calls before any stream capture).  Calls share the
 * array: calls that overlap on the GPU race -- keep them on one stream. */
#define THR_NOALLOC_MAX_CTAS 4096
int thr_sum_f32_noalloc(uint64_t x, uint64_t n, uint64_t out, uint32_t ctas, uint64_t stream);

/* Peer mailboxes for the in-kernel combine of a sharded sum (one process per
 * GPU).  No counterpart in the reference, whose multi-GPU step is an NCCL
 * all-reduce of the per-GPU partials; this replaces that all-reduce with
 * stores over NVLink from inside the reduction kernel.
 *   thr_peer_alloc: a zeroed device buffer of `bytes` on the current device
 *     and its CUDA IPC handle (64 bytes) for the other processes;
 *   thr_peer_open:  map another process's buffer from its handle (peer
 *     access enabled lazily); thr_peer_close unmaps it;
 *   thr_peer_free:  release a buffer made by thr_peer_alloc.
 * Plain cudaMalloc device memory, not bound to any NVLink switch object. */
#define THR_IPC_HANDLE_BYTES 64
int thr_peer_alloc(uint64_t bytes, uint64_t *dptr, unsigned char handle[THR_IPC_HANDLE_BYTES]);
int thr_peer_open(const unsigned char handle[THR_IPC_HANDLE_BYTES], uint64_t *dptr);
int thr_peer_close(uint64_t dptr);
int thr_peer_free(uint64_t dptr);

#ifdef __cplusplus
}
#endif

#endif /* THOMPILER_RUNNER_H */
