/*
 * C ABI of the B200 (sm_100a) quantized matvec / matmul library: libint4matmul_b200.so.
 *
 * This is the boundary a foreign-function binding attaches to.  Everything is plain pointers and
 * sizes; all data pointers are DEVICE pointers on the current CUDA device; nothing here allocates
 * device memory unless the entry says so (only i4mm_peer_buffer_create does); every launch goes onto the stream passed in (a
 * cudaStream_t cast to void*, NULL = the legacy default stream the reference launches on).
 * Calls return an i4mm_status; they never abort the process and never trap the device.
 *
 * Tensor contract (identical to the reference's torch extension, int4matmul.cpp:26-48):
 *   x       fp16  (rows, N)          rows = B*M flattened, N = in-features (reduction dim)
 *   matrix  int32 (R, S)             packed weights, S = out-features contiguous;
 *                                    dense: R = N*bits/32; 16:32 sparse int4: R = N/16
 *   mask    int32 (N/32, S) or NULL  16:32 keep-mask, bit l of [b, s] = keep(n = 32b+l, s)
 *   scales  fp16  (n_groups, S)      scale >= 0: W = (q - zero) * scale, both steps rounded to fp16
 *   zeros   fp16  (n_groups, S)      scale <  0: W = fma(+-2^(q & (2^(bits-1)-1)), -scale, zero)
 *                                    Any zero-point is exact.  The fastest decode takes scales >= 0 with integer zero-points
 *                                    0 .. 512 (16:32: 0 .. 127).  With others up to about 128 rows take up to 1.6 times as long (one
 *                                    row 16384^2: int4 35 and 52 us; 16:32 51 and 78, with integers up to 255 67), with scales < 0
 *                                    up to twice (every second group: 70 and 94); 512 rows int4 1.1 and 3 times.
 *   out     fp16  (rows, S)
 *   group_size  positive multiple of 64, or negative for "one group over all of N"
 *   N, S multiples of 64.  sparse is only defined for bits == 4.
 */
#ifndef INT4MATMUL_B200_H
#define INT4MATMUL_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum i4mm_status {
    I4MM_OK = 0,
    I4MM_ERR_BITS = 1,         /* bits not in {4, 3, 2}          (int4matmul.cpp:35, 45) */
    I4MM_ERR_UNSUPPORTED = 2,  /* sparse with int3 / int2         (matmul.cuh:188, 331 trap in the reference) */
    I4MM_ERR_SHAPE = 3,        /* a size rule of matmul_kernel.cu:383, 404-416 is violated */
    I4MM_ERR_NULL = 4,         /* a required pointer is NULL */
    I4MM_ERR_ALIGN = 5,        /* a pointer is not 16-byte aligned */
    I4MM_ERR_WORKSPACE = 6,    /* workspace missing or smaller than i4mm_workspace_bytes() */
    I4MM_ERR_LAUNCH = 7,       /* CUDA reported an error at launch; see i4mm_last_cuda_error() */
    I4MM_ERR_MASK = 8,         /* a 32-block of the keep-mask does not hold exactly 16 entries */
    I4MM_ERR_DEVICE = 9,       /* device is not sm_100 or a driver entry point is unavailable */
    I4MM_ERR_TIMEOUT = 10,     /* a bounded device-side wait gave up (status word set by the kernel) */
    I4MM_ERR_TOO_LARGE = 11    /* the problem exceeds the fixed scratch of i4mm_quant_matvec_static */
} i4mm_status;

/* Human-readable name of a status code. */
const char* i4mm_status_string(int status);
/* The cudaError_t (as int) recorded by the last call that returned I4MM_ERR_LAUNCH on this thread. */
int i4mm_last_cuda_error(void);
/* Library version: major*10000 + minor*100 + patch. */
int i4mm_version(void);
/* Kernels this library has launched in this process so far, over all entry points (a multiply is one launch,
 * or two where it cuts K into parts and reduces them).  For accounting in benchmarks; no reference counterpart. */
unsigned long long i4mm_launch_count(void);
/* What the last i4mm_quant_matmul call of this host thread launched: on the tcgen05 path the rows per tile (the MMA's N:
 * 16, 32, 64, 128, 160, 192, 224 or 256) + 1000 if it ran as CTA pairs + 10000 * K parts; 8 after a call that took the
 * few-row kernel (up to 8 rows of a small matrix, path 0); 0 after a call that took the streaming path.  For tests that
 * must know which kernel instance they exercised; no reference counterpart. */
int i4mm_last_launch_shape(void);
/* How that launch spread the work over the GPU: 0 not the tcgen05 path; whole tiles of the shapes that are made for them; K parts (a
 * second kernel adds them); or the weight-streaming shape (any row count up to 64, tiles of 128 rows above) with equal ranges of units
 * for all CTAs, with whole tiles, or with the same number k of CTAs for every tile (I4MM_SCHEDULE_STREAM_CTAS_PER_TILE + k). */
#define I4MM_SCHEDULE_WHOLE_TILES 1
#define I4MM_SCHEDULE_K_PARTS 2
#define I4MM_SCHEDULE_STREAM_EQUAL_RANGES 3
#define I4MM_SCHEDULE_STREAM_WHOLE_TILES 4
#define I4MM_SCHEDULE_STREAM_CTAS_PER_TILE 1000
int i4mm_last_launch_schedule(void);

/*
 * Bytes of device scratch the two multiply entries need.  The scratch holds the per-CTA partial tiles
 * of the split-K reduction (on the tcgen05 and few-row paths words that tell by themselves that they have been
 * written, on the streaming path with arrival counters), a word per CTA and a status word.  It must be zero-filled once
 * before its first use; the kernels leave it all-zero again when they finish, so one buffer can serve every later call on
 * the same stream.
 * Calls that overlap on the device must not share a buffer.  After a call for which
 * i4mm_device_status reported I4MM_ERR_TIMEOUT, zero the buffer again before reusing it.
 */
size_t i4mm_workspace_bytes(void);

/*
 * out[r, s] (+)= sum_n x[r, n] * W16[n, s], fp32 accumulation, one rounding to fp16.
 *
 * Replaces matvec_packed_int<bits> / MVA_Int4_Half (matvec_kernel.cu:302-383, 198-267) and
 * matmul_packed_int<bits> / MMA_Int4_Half (matmul_kernel.cu:375-459, 219-333).
 *
 *   accumulate != 0  ->  out = half(float(out) + x.W): what the reference's matvec route does to the
 *                        caller's `outs` (matvec_kernel.cu:351, 263, 381-382)
 *   accumulate == 0  ->  out is overwritten, as the reference's matmul route does (matmul_kernel.cu:299-332)
 *
 * A multiply gets through on however few SMs the kernels of other streams leave it, with the same result: no block waits for
 * one that the GPU starts after it (blocks start in the order of their numbers), or gives that up after ~0.15 ms.
 *
 * rows = B*M may be any value >= 0 (rows == 0 returns I4MM_OK without a launch).  The entry picks the few-row kernel
 * for up to 8 rows of a small matrix and the tcgen05 tensor-core kernel for everything else; `path` forces one:
 *   0 = automatic (the streaming kernel where the driver's tensor-map encoder is not found), 1 = streaming (mma.sync,
 *   split-K over the whole GPU), 2 = tcgen05 / TMEM pipeline (128 rows or more run as CTA pairs, two SMs per
 *   MMA), 3 = tcgen05 with single CTAs only.
 *   With path 2 or 3, `path | (T << 8)` also fixes the rows per tile (the MMA's N) to T in {16, 32, 64, 128, 160, 192,
 *   224, 256} instead of choosing it by shape (T >= 128 with path 2 runs as CTA pairs; T <= 64 needs rows <= T):
 *   for tests and tuning, results do not depend on it beyond fp32 summation order.
 *   `path | I4MM_PATH_STATIC_WEIGHTS` is the caller's promise that matrix, mask, scales and zeros are not written by
 *   the kernel that precedes this call in the stream (weights of a loaded model never are).  Launches may begin while
 *   that kernel is still finishing (programmatic dependent launch); with the promise the first weight copies go out
 *   then, while x, out and the workspace are touched only once that kernel is complete.  Without it nothing at all is
 *   read before, as with the reference's launches.  The kernels of this library let their successor begin only once
 *   everything before them is complete, so the promise is about one kernel; a row norm that carries the same flag is the
 *   exception (see i4mm_row_norm).
 */
#define I4MM_PATH_STATIC_WEIGHTS 0x100000
int i4mm_quant_matmul(int bits, int accumulate, int path,
                      void* out, const void* matrix, const void* mask /* NULL = dense */,
                      const void* x, const void* scales, const void* zeros,
                      int64_t rows, int64_t N, int64_t S, int64_t n_groups, int64_t group_size,
                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * The multiply of one rank of a column-sharded matrix, with the all-gather of the outputs done by the kernel's own
 * stores.  No counterpart in the reference (which has no multi-GPU code); it serves the layer-stack configuration,
 * where every matrix is sharded along S over the GPUs of one node and the next matrix needs all of S.
 *
 *   matrix, mask, scales, zeros   this rank's shard: S columns = `parts` pieces of S / parts columns each, piece j being
 *                                 this rank's columns of the j-th matrix of a concatenation (q | k | v, gate | up; 1 = one matrix)
 *   gathered[0 .. n_gathered)     (rows, ld) fp16 buffers, normally one per rank (this rank's own and the peers', opened
 *                                 with i4mm_peer_buffer_open); the result is stored into every one of them, local column
 *                                 c of piece j at column j * (S / parts) * world + rank * (S / parts) + c
 *   ld >= S * world, a multiple of 8.  Always overwrites (no accumulate); tcgen05 kernel only (path 0, 2 or 3).
 * The stores are plain global stores through the peer mappings; i4mm_gather_sync afterwards tells the peers and waits
 * for them.  A buffer may be written again only after another i4mm_gather_sync has passed since its readers ran.
 */
int i4mm_quant_matmul_gather(int bits, int path, void* const* gathered, int n_gathered, int64_t ld, int64_t parts,
                             int64_t rank, int64_t world, const void* matrix, const void* mask /* NULL = dense */,
                             const void* x, const void* scales, const void* zeros,
                             int64_t rows, int64_t N, int64_t S, int64_t n_groups, int64_t group_size,
                             void* workspace, size_t workspace_bytes, void* stream);

/*
 * Device buffers that other processes of the node can map (CUDA IPC), for i4mm_quant_matmul_gather.
 *   create   cudaMalloc + zero-fill + export: *dev_ptr = the buffer, handle_out = i4mm_ipc_handle_bytes() bytes to send to the peers
 *   open     map a peer's buffer from its handle (peer access is enabled on first use); close unmaps it
 *   destroy  frees a buffer made by create (after the peers have closed it)
 * These four and nothing else in the library allocate or free device memory.
 */
size_t i4mm_ipc_handle_bytes(void);
int i4mm_peer_buffer_create(size_t bytes, void** dev_ptr, void* handle_out);
int i4mm_peer_buffer_open(const void* handle, void** dev_ptr);
int i4mm_peer_buffer_close(void* dev_ptr);
int i4mm_peer_buffer_destroy(void* dev_ptr);

/*
 * Hand-shake after a gathering multiply.  Every rank has a flags buffer of i4mm_gather_flags_bytes(slots) bytes made
 * with i4mm_peer_buffer_create (zero-filled) and opened by the peers; flags[r] = rank r's buffer as seen from here
 * (flags[rank] = the local one).  The call enqueues one small kernel that, for slot `slot` (one slot per gathered
 * buffer that is in flight at a time), tells every rank that this rank's stores are done and waits until every rank has
 * said the same.  All ranks must issue the same sequence of calls.  The values exchanged advance by themselves on the
 * device, so the call can be captured in a CUDA graph and replayed.  The wait is bounded (about two seconds): a peer
 * that never arrives sets the status word of `workspace` (see i4mm_device_status) instead of hanging the GPU.
 */
size_t i4mm_gather_flags_bytes(int64_t slots);
int i4mm_gather_sync(void* const* flags, int64_t world, int64_t rank, int64_t slot, int64_t slots, void* workspace, void* stream);

/*
 * The same multiply as i4mm_quant_matmul on its streaming path, for callers that cannot allocate device
 * memory (no cudaMalloc available to them: code running inside someone else's memory pool, inside a
 * latency-critical loop where an allocation would synchronise the device, or in a sandbox that only hands out
 * buffers registered up front).  The caller passes inputs and outputs as usual and NO workspace: the split-K
 * scratch is a fixed 4 882 688-byte array inside the library image, held by every GPU context that loads the
 * library until the process exits.  This entry has no counterpart in the reference.
 *
 *   limits   rows <= 8 and S <= 1 048 576; anything larger returns I4MM_ERR_TOO_LARGE and launches nothing
 *   set-up   the first call on each device looks up the array's device address (cudaGetSymbolAddress) and
 *            configures the kernel; make that first call before any stream capture begins
 *   sharing  every call on a device uses the same array, which keeps the previous call's contents; the entry
 *            clears the counters it needs (one small memset on `stream`) before launching.  Two calls that
 *            overlap on the GPU (different streams, or different host threads) race on it: serialise them.
 *   It calls no cudaMalloc, cudaFree or any allocating library routine.  Results are identical to
 *   i4mm_quant_matmul(path = 1) on the same inputs.
 */
int i4mm_quant_matvec_static(int bits, int accumulate,
                             void* out, const void* matrix, const void* mask /* NULL = dense */,
                             const void* x, const void* scales, const void* zeros,
                             int64_t rows, int64_t N, int64_t S, int64_t n_groups, int64_t group_size, void* stream);

/*
 * Waits for the stream and reports whether a kernel that used `workspace` gave up on one of its bounded
 * device-side waits (every wait on a shared-memory barrier inside the kernels has a poll limit, after which
 * the kernel records a status word in the workspace and returns instead of spinning).  Returns I4MM_OK, or
 * I4MM_ERR_TIMEOUT after clearing the word.  No counterpart in the reference, whose kernels have no waits.
 */
int i4mm_device_status(void* workspace, void* stream);
/* The same check for i4mm_quant_matvec_static, whose status word lives in the library's fixed scratch on the
 * current device: waits for the stream, returns I4MM_OK or (after clearing the word) I4MM_ERR_TIMEOUT. */
int i4mm_static_device_status(void* stream);
/*
 * Scratch whose first use comes while a stream is being captured into a CUDA graph has to be allocated, zero-filled and waited for outside
 * of the graph: as nodes of it, the zero-filling would be repeated at every replay, and missing where another graph that shares the
 * scratch is replayed first.  A thread may do that during a capture if its capture mode is relaxed.  Sets the calling thread's mode to *mode
 * (0 global, 1 thread-local, 2 relaxed) and leaves the former one there, as cudaThreadExchangeStreamCaptureMode does.
 */
int i4mm_exchange_capture_mode(int* mode);

/*
 * 16:32 packer.  Replaces sparse_int4_pack / PackMatrix (utils_kernel.cu:67-119, 19-64).
 *   wt_in, msk_in  uint8 (S, N): low nibble of wt_in is the weight, msk_in > 0 means keep
 *   wt_out int32 (N/16, S), msk_out int32 (N/32, S)
 *   violations     optional device int32; incremented once per 32-block that does not keep exactly
 *                  16 entries (the reference device-asserts instead, utils_kernel.cu:41).  May be NULL.
 */
int i4mm_sparse_pack(void* wt_out, void* msk_out, const void* wt_in, const void* msk_in,
                     int64_t S, int64_t N, void* violations, void* stream);

/*
 * Counts the 32-blocks of an already packed keep-mask (N/32, S) whose popcount is not 16 into the
 * device int32 *violations (which the caller zeroes).  No counterpart in the reference, which trusts
 * the mask; offered so callers can validate foreign masks without a device trap.
 */
int i4mm_check_mask(const void* mask, int64_t N, int64_t S, void* violations, void* stream);

/*
 * Row-wise glue of the layer-stack runner: y[r, :] = v / rms(v) per row, computed in fp32, with
 *   mode 0: v = a     mode 1: v = a + b + c     mode 2: v = a + b / rms(b)     mode 3: v = a * b
 *   mode 4: mode 2 into y[0 : rows*width], then mode 0 of that (rounded) result into y[rows*width : 2*rows*width]
 *           (a layer's residual stream and the next layer's normalised input from one launch)
 * a, b, c fp16 (rows, width) with row strides in elements (column slices of a gathered buffer are fine);
 * y fp16 (rows, width) contiguous ((2, rows, width) in mode 4); width even; pointers 4-byte aligned.  No counterpart in the reference
 * (it has no model code): it replaces the handful of eager elementwise kernels between two quantized linears.
 * `mode | I4MM_PATH_STATIC_WEIGHTS` extends the promise of that name: the kernel that precedes the row norm (and those before
 * it, as long as they are row norms with this flag too) does not write weight-side tensors of the multiply after it either.
 * That multiply, if it carries the promise itself, may then copy weights while the kernel before the row norm is running.
 */
int i4mm_row_norm(int mode, void* y, const void* a, const void* b, const void* c, int64_t rows, int64_t width,
                  int64_t stride_a, int64_t stride_b, int64_t stride_c, void* stream);

/*
 * ---- paged key-value cache in 8 bits ------------------------------------------------------------------------------
 * What stands between the quantized linears of a decoder that generates text: the keys and values of all tokens so far, in
 * pages of 16, 32, 64 or 128 tokens, 8 bits a value with one scale for each page and head, and the attention over them.  No
 * counterpart in the reference, which has no model code.
 *
 *   k, v      (pages, heads, page_size, head_dim) int8 or e4m3 (1 byte a value), head_dim 64 or 128 and contiguous; the other strides
 *             are free (multiples of 16 bytes, below 2^31).  Here and for activations, the stride of a dimension of size 1 may be anything
 *   scales    fp32 (pages, heads, 2) contiguous, 8-byte aligned: of the page's keys and of its values.  A byte q stands for q * scale.
 *   slot      where a token lies: page * page_size + place in the page.  Slots outside of the cache (negative ones: padding) are
 *             skipped by the writer and read as zeros.
 *   block_table   int32 (requests, table_width): page j of a request holds its tokens j * page_size and on.  Entries outside of
 *             [0, pages) are no pages: attention sees no tokens there.
 * Lengths, slots and page numbers are int32; activations are fp16 (type 0) or bf16 (type 1).
 */
#define I4MM_CACHE_INT8 0
#define I4MM_CACHE_E4M3 1
#define I4MM_TYPE_FP16 0
#define I4MM_TYPE_BF16 1
typedef struct i4mm_cache {
    void* k;
    void* v;
    void* scales;
    int64_t pages, heads, page_size, head_dim;
    int64_t k_page_stride, k_head_stride, k_token_stride;    /* bytes (= values) */
    int64_t v_page_stride, v_head_stride, v_token_stride;
    int32_t type;                                            /* I4MM_CACHE_INT8 or I4MM_CACHE_E4M3 */
} i4mm_cache;

/*
 * The tables of one step, from the requests' lengths, in one launch.
 *   seq_lens (requests)     tokens held before the step            new_lens (requests)   tokens that it adds; negative: the request ends,
 *                                                                                        its pages are free again and its length is 0
 *   block_table             entries of the pages that the step begins are written in place (row stride in entries)
 *   free_pages (capacity)   a stack: entries [0, *free_count) are free.  The pages of the requests that end are pushed in request order,
 *                           then new pages are taken off its top in request order; where none is left the entry becomes -1
 *   outputs                 lens_after (requests); cu_lens (requests + 1): the packed place of each request's first new token;
 *                           slots, positions, request_of (max_tokens): of every packed token, -1 beyond the last one and, for slots, where
 *                           there is no page; counts (2): *free_count afterwards, and the number of pages that could not be had
 *                           (the stack was empty, or the table's row full)
 * seq_lens, new_lens and free_count are left alone, so that the same call again gives the same answers; free_count is not one of the
 * outputs.  Where counts[1] is not 0 the step had better be dropped, and a smaller one made from the same lengths and count: a request
 * that went on without its pages would give -1 back as pages when it ends.  requests <= 16384, requests * table_width and max_tokens
 * <= 2^30; packed tokens beyond max_tokens get no entry.
 */
int i4mm_cache_plan(int64_t requests, const void* seq_lens, const void* new_lens, void* block_table, int64_t table_width,
                    int64_t table_stride, void* free_pages, int64_t free_capacity, const void* free_count, int64_t page_size,
                    int64_t max_tokens, void* lens_after, void* cu_lens, void* slots, void* positions, void* request_of, void* counts,
                    void* stream);

/*
 * Quantises k and v (tokens, heads, head_dim; strides in elements) into the cache at `slots`.
 * The tokens of one page that a call writes are neighbours in the call, with ascending slots (as i4mm_cache_plan lays them out); the
 * places of the page before the first of them hold tokens already, or the first of them is the page's first and what the page held is void.
 * With a = the largest finite |value| that a call adds to a page and head and `most` = 127 or 448, the scale becomes the larger of the old
 * one and the least power of two s (2^-100 at least) with a <= most * s, 0 for a = 0, the new bytes are round(x / s), and if the scale grew the bytes already there
 * become round(q * old / s).  Since scales grow by powers of two, a value is off by less than one step of its final scale however often
 * that happens (1/2 + 1/4 + ...).  Infinities are stored as +-most, NaN as 0.
 */
int i4mm_cache_write(const i4mm_cache* cache, const void* k, const void* v, int type, int64_t tokens, int64_t k_token_stride,
                     int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const void* slots, void* stream);

/* The values at `slots`: k_out, v_out (tokens, heads, head_dim) contiguous.  Exact where the scales are powers of two. */
int i4mm_cache_read(const i4mm_cache* cache, void* k_out, void* v_out, int type, int64_t tokens, const void* slots, void* stream);

/*
 * out[t, h, :] = sum_j w_j v_j,  w = softmax over the tokens j that row t sees of scale * q[t, h, :] . k_j
 *   q (tokens, q_heads, head_dim), strides in elements; out the same, contiguous; q_heads a multiple of the cache's heads: query head h
 *   reads head h / (q_heads / heads)
 *   seq_lens (requests)       tokens in the cache, those of this step included
 *   cu_lens (requests + 1)    rows of request b are cu_lens[b] .. cu_lens[b + 1] (NULL: one row for each request), its last ones: row i of
 *                             n is at position p = seq_lens[b] - n + i and sees the tokens j <= p, with window > 0 those with
 *                             j > p - window.  Rows that see no token, and rows of no request, are 0.
 *   table_width               a row of the block table stands for table_width * page_size tokens, at most 2^31 - 128
 *   max_len                   the most rows of a request, for the choice of a kernel (a wrong one costs time, nothing else)
 * Sums and softmax statistics are fp32.  Which kernel runs goes by sizes that the host has (rows, max_len, the table's width, window), and the two
 * round differently: the one for few rows multiplies the values by weights of about 22 bits, the one for prompts by weights rounded to fp16
 * (2^-11 of each; against 64 bits 2.6e-4 to 2.8e-4 of an fp16 output's norm, where rounding the output alone makes 2.1e-4).  The same call gives the same bits.  `workspace` (about 65 MB): i4mm_cache_attention_workspace_bytes() bytes, zero-filled before the first use
 * and after i4mm_device_status has reported I4MM_ERR_TIMEOUT for it, shared by calls of one stream only
 * (made by any number of host threads: calls with one workspace launch their kernels one call after the other).
 */
size_t i4mm_cache_attention_workspace_bytes(void);
int i4mm_cache_attention(const i4mm_cache* cache, void* out, const void* q, int type, int64_t tokens, int64_t q_heads,
                         int64_t q_token_stride, int64_t q_head_stride, const void* block_table, int64_t table_width,
                         int64_t table_stride, const void* seq_lens, const void* cu_lens, int64_t requests, int64_t max_len, float scale,
                         int64_t window, void* workspace, size_t workspace_bytes, void* stream);
/* The kernels that the last i4mm_cache_attention call of this host thread launched, or-ed; 0: none (an empty or a refused call).  For tests
 * that must know which kernel they exercised. */
#define I4MM_ATTENTION_FEW_ROWS 1
#define I4MM_ATTENTION_PROMPT 2
#define I4MM_ATTENTION_PREFIX 4           /* prefixes that few rows read */
#define I4MM_ATTENTION_MANY_READERS 8     /* prefixes that many rows read */
int i4mm_last_attention_kernels(void);

/*
 * angles[t, i] = (cos, sin) of positions[t] * freqs[i], fp32 (tokens, pairs, 2) contiguous; (1, 0) where the position is negative (padding).
 *   positions int32 (tokens), freqs fp32 (pairs), pairs a multiple of 8 up to 128; angles 16-byte, freqs 8-byte aligned.
 * The products and their reduction by whole turns are fp64: the angle is off by at most 9.4e-8 (its rounding to fp32 after that) and 2^-51 of itself,
 * 1.5e-7 for 2^27 radians and 1.1e-6 for 2^31.
 */
int i4mm_cache_angles(void* angles, const void* positions, const void* freqs, int64_t tokens, int64_t pairs, void* stream);

/*
 * i4mm_cache_write for a model whose queries and keys are normed and rotated, in the same launch.  For each row x (head_dim values) of a head of q or k:
 *   y = x / sqrt(mean(x^2) + eps) * weight     (q_weight, k_weight: (head_dim) in the activations' type, 16-byte aligned; NULL: y = x)
 *   (a, b) -> (a cos - b sin, b cos + a sin)   of the first 2 * pairs values, a and b being values i and i + pairs, or with pairs_beside 2 i and 2 i + 1;
 *                                              cos, sin = angles[t, i] (fp32 (tokens, pairs, 2), 16-byte aligned); pairs a multiple of 8, 0: no rotation
 * in fp32, rounded once to the activations' type.  q_out (tokens, q_heads, head_dim) contiguous gets the queries of all tokens; the keys, and
 * the values as they are, go into the cache as i4mm_cache_write's do, to the byte.  q_out is none of the inputs; q_heads is free here.  With neither
 * weights nor pairs it is a write that also copies the queries.
 */
int i4mm_cache_append(const i4mm_cache* cache, void* q_out, const void* q, const void* k, const void* v, int type, int64_t tokens, int64_t q_heads,
                      int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                      int64_t v_head_stride, const void* slots, const void* angles, int64_t pairs, int pairs_beside, const void* q_weight,
                      const void* k_weight, float eps, void* stream);

/*
 * Shared prefixes: requests that begin alike hold what they share once.  A prefix is a place of the batch like any request (its tokens are
 * written, and its pages given back, as theirs are); a request names it and holds only what comes after it.
 *   prefix_of (requests)      the place whose tokens come before the request's own.  None: negative, no place of the batch, the request itself, a
 *                             place without tokens; a prefix's own prefix is not looked at.  Positions behind a place count its tokens: where keys
 *                             are rotated it must not grow any more.
 *   seq_lens, cu_lens         as for i4mm_cache_attention, after the step
 * Outputs: effective (requests): prefix_of, -1 for none; starts (requests + 1), rows (max_tokens): the packed rows that read place p are
 * rows[starts[p]] .. rows[starts[p + 1] - 1], ascending, -1 behind the last of all; positions (max_tokens): of the packed rows, the prefix counted
 * (for i4mm_cache_angles), -1 for padding.  requests <= 16384, max_tokens <= 2^30.
 */
int i4mm_cache_share(int64_t requests, const void* prefix_of, const void* seq_lens, const void* cu_lens, int64_t max_tokens, void* effective,
                     void* starts, void* rows, void* positions, void* stream);

/*
 * i4mm_cache_attention of rows that see their request's prefix before its own tokens: with L tokens in the prefix, a row at position p of its request
 * (p >= 0) sees tokens j of the prefix and j' <= p of its own; with window > 0 those with j > L + p - window and j' > p - window.  The prefix's pages
 * are fetched and decoded once for every 64 rows of a key head (readers times q_heads / heads), once for every 256 where there are more than 256.
 *   prefix_of, prefix_starts, prefix_rows (listed >= tokens entries)   i4mm_cache_share's effective, starts and rows of the same step
 *   scratch   i4mm_cache_shared_scratch_bytes(tokens, q_heads, head_dim) bytes (4 a value of q and 8 a row and head, whichever rows have a prefix),
 *             16-byte aligned, of any contents, this call's alone.  What it held
 *             counts for rows whose request names a prefix and which no list names (lists of another step): their results are void, but nothing
 *             beyond the arrays is read for them
 * heads * (table_width * page_size / 128 + 5) * (tokens * (q_heads / heads) / 64 + the smaller of requests and tokens) has to be below 2^31
 * (I4MM_ERR_TOO_LARGE otherwise).  In a step of no requests the tables are not looked at.  The prefix's sums are fp32 too, its weights rounded to fp16;
 * everything else is as above.
 */
size_t i4mm_cache_shared_scratch_bytes(int64_t tokens, int64_t q_heads, int64_t head_dim);
int i4mm_cache_attention_shared(const i4mm_cache* cache, void* out, const void* q, int type, int64_t tokens, int64_t q_heads,
                                int64_t q_token_stride, int64_t q_head_stride, const void* block_table, int64_t table_width,
                                int64_t table_stride, const void* seq_lens, const void* cu_lens, int64_t requests, int64_t max_len, float scale,
                                int64_t window, const void* prefix_of, const void* prefix_starts, const void* prefix_rows, int64_t listed,
                                void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* INT4MATMUL_B200_H */
