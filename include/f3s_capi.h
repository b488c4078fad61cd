/*
 * f3s_capi.h -- C-ABI of libf3s_hip.so, the MI355X (gfx950) implementation of
 * the fused3S hot path: CSR -> 16x16 block-sparse conversion, window ordering
 * and the fused SDDMM -> online softmax -> SpMM pass.
 *
 * Plain C: no HIP or torch types.  Device buffers are `void*`/typed pointers
 * obtained from f3s_malloc (or any HIP allocation in the same process);
 * streams are `void*` (a hipStream_t, NULL = the default stream).  Every
 * function returns f3s_status (0 = F3S_OK) and never exits the process; the
 * detail of the last failure on the calling thread is f3s_last_error().
 *
 * Layouts:
 *   CSR            row_ptr int32[n+1], col_idx int32[nnz] (columns < n)
 *   block-sparse   W = ceil(n/16) row windows; window_offsets int32[W+1];
 *                  block_col int32[T] (ascending per window);
 *                  tile_mask uint16[T][16]: bit c of row r <=> edge
 *                  (16w + r, 16*block_col + c)
 *   features       Q, K, V: IEEE binary16 bits, node-major [n][H][d];
 *                  O: float32 [n][H][d].  Buffers need n rows (a reference-
 *                  style buffer padded to 16W rows also works).
 *
 * Thread safety: calls on different streams may run concurrently; the
 * library's only mutable global state is the per-thread last error and the
 * per-device cache of freed device memory (below; one mutex guards it).
 * A plan owns the partial-result buffers of its split windows, so one plan
 * must not serve two overlapping calls.
 */
#ifndef F3S_CAPI_H
#define F3S_CAPI_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef int32_t f3s_status;

#define F3S_OK 0
#define F3S_EINVAL 1        /* bad size, pointer or argument */
#define F3S_ENOMEM 2        /* device allocation failed */
#define F3S_EHIP 3          /* a HIP runtime call failed (detail in f3s_last_error) */
#define F3S_ENODEV 4        /* no usable GPU */
#define F3S_EUNSUPPORTED 5  /* valid but not implemented here (e.g. d != 64) */
#define F3S_EDATA 6         /* input data violates the format (e.g. column >= n) */

#define F3S_ABI_VERSION 1

/* 16-bit types of the calls that take both. */
#define F3S_F16 0           /* IEEE binary16 */
#define F3S_BF16 1          /* bfloat16 */

/* Semantics of f3s_attention_fwd*: tile_mask == NULL selects TILE_DENSE
 * (every column < n of every active tile is attended: the reference kernel
 * and test ground truth, tests/test_fused_3s_v2.cu:17-59); a mask selects
 * MASKED (edge-exact, baselines/cpu_baseline.cpp:16-91). */

const char* f3s_status_string(f3s_status s);
const char* f3s_last_error(void);
int32_t f3s_abi_version(void);

/* Loads the library's GPU code onto the current device now rather than at
 * the first launch of each kernel (HIP loads code objects lazily), so the
 * first timed call is not charged for it.  Optional; idempotent.  The
 * reference has no counterpart (CUDA contexts load modules the same way). */
f3s_status f3s_init(void);

/* ---- device plumbing (replaces the CUDA_CHECK'ed runtime calls of the
 *      reference harness, tests/test_fused_3s_v2.cu:93-120,139,157-159) ---- */
f3s_status f3s_device_count(int32_t* count);
f3s_status f3s_set_device(int32_t device);
f3s_status f3s_device_name(char* buf, int32_t buflen);
/* Device memory comes from a caching allocator over hipMalloc: blocks the
 * library frees (scratch of a call, in stream order; a destroyed plan's
 * buffers) are kept per device and size class for reuse, so repeated
 * conversions, plans and calls skip the driver's allocation and page
 * mapping.  Idle cached memory is capped per device at 1 GiB, or at the
 * F3S_CACHE_LIMIT_MB environment variable's value read at the first
 * allocation (0 keeps nothing); on an allocation failure the cache goes back
 * to the driver and the allocation is retried.  f3s_malloc'd memory is usable
 * on every stream on return; f3s_free waits for the device first, as hipFree
 * does, and returns the block to the cache (f3s_release_cached_memory hands
 * every idle block back to the driver). */
f3s_status f3s_malloc(void** ptr, uint64_t bytes);
f3s_status f3s_free(void* ptr);
/* Returns every idle cached block to the driver (waits for every device
 * first).  No reference counterpart; for processes that share the GPU with
 * another allocator, e.g. torch's. */
f3s_status f3s_release_cached_memory(void);
f3s_status f3s_memcpy_h2d(void* dst, const void* src, uint64_t bytes, void* stream);
f3s_status f3s_memcpy_d2h(void* dst, const void* src, uint64_t bytes, void* stream);
f3s_status f3s_memcpy_d2d(void* dst, const void* src, uint64_t bytes, void* stream);
f3s_status f3s_memset(void* ptr, int32_t value, uint64_t bytes, void* stream);
f3s_status f3s_synchronize(void* stream);            /* NULL: whole device */
f3s_status f3s_stream_create(void** stream);
f3s_status f3s_stream_destroy(void* stream);
f3s_status f3s_event_create(void** event);
f3s_status f3s_event_destroy(void* event);
f3s_status f3s_event_record(void* event, void* stream);
f3s_status f3s_event_elapsed_ms(void* start, void* stop, float* ms);  /* waits for stop */

/* float2half_kernel (tests/test_fused_3s_v2.cu:61-64): IEEE round to
 * nearest even, elementwise. */
f3s_status f3s_cast_f32_to_f16(const float* d_in, uint16_t* d_out, int64_t count, void* stream);

/* convert_csr_to_block_sparse (src/converter.cu:13-44), on the GPU.
 * d_window_offsets[W+1] is always written and *T_out receives T (the call
 * synchronises `stream` to read it).  When d_block_col is non-NULL the tile
 * lists are written too (it must hold T entries), and when d_tile_mask is
 * non-NULL the 16 row masks of each tile (T*16 entries).  Typical use is two
 * calls: sizes first (d_block_col = NULL), then the lists.  Output is
 * bit-exact with the reference converter.  F3S_EDATA if row_ptr is not
 * monotone from 0 to nnz or a column is outside [0, n) (the offsets written
 * are then meaningless).  A CSR may repeat an entry (a multigraph): the
 * reference converter accepts that, and so does this one -- the tile lists
 * are those of the deduplicated CSR and the masks record each (row, column)
 * pair once, so nnz - mask_bits (f3s_bsf_stats) counts the repeated entries.
 * The masked pass then attends each edge once, whereas the reference's
 * cpu_sparse_attention_csr (baselines/cpu_baseline.cpp:38-50) counts a
 * repeated entry once per repeat; the tile-dense pass is unaffected.  Each
 * call makes one host round trip (to read T and the error bits); scratch
 * comes from the library's cache. */
f3s_status f3s_convert_csr_to_bsf(const int32_t* d_row_ptr, const int32_t* d_col_idx,
                                  int32_t n, int64_t nnz,
                                  int32_t* d_window_offsets, int32_t* d_block_col,
                                  uint16_t* d_tile_mask, int64_t* T_out, void* stream);

/* Count and fill in one call and one host round trip (no reference
 * counterpart): block_col and tile_mask (NULL: no masks) hold min(nnz, W * W)
 * entries, W = ceil(n / 16), which T never exceeds; the first T are written.
 * n up to 4,194,304.  Errors as of the two calls. */
f3s_status f3s_convert_csr_to_bsf_once(const int32_t* d_row_ptr, const int32_t* d_col_idx,
                                       int32_t n, int64_t nnz, int32_t* d_window_offsets,
                                       int32_t* d_block_col, uint16_t* d_tile_mask,
                                       int64_t* T_out, void* stream);

/* generate_balanced_window_order (include/utils.cuh:48-59), on the GPU:
 * windows by descending tile count, ties by ascending window index. */
f3s_status f3s_window_order(const int32_t* d_window_offsets, int32_t W,
                            int32_t* d_order, void* stream);

/* Figures behind the algorithmic byte model (no reference counterpart):
 * occ_sum = sum over tiles of the columns the fused pass gathers (popcount of
 * the OR of the row masks if d_tile_mask, else the tile's columns < n);
 * mask_bits = popcount of all masks, the distinct edges: mask_bits < nnz iff
 * the CSR repeats entries.  Synchronises `stream`. */
f3s_status f3s_bsf_stats(const int32_t* d_block_col, const uint16_t* d_tile_mask,
                         int64_t T, int32_t n, int64_t* occ_sum, int64_t* mask_bits,
                         void* stream);

/* f3s_1tb1rw_kernel (src/fused3s_v2.cu:81-90) and its launch
 * (tests/test_fused_3s_v2.cu:124-131): one fused pass, each row window
 * handled whole, over the windows d_window_order names (NULL = all).
 * O[i] = sum_j softmax_j(scale * Q[i].K[j]) V[j] per head; rows with no
 * attended column get 0; rows of windows the order does not name are not
 * written.  Requires d == 64 and 1 <= H <= 64 heads in node-major [n][H][64]
 * layout, of any size (tensors past ~4 GiB are read with 64-bit addresses);
 * scale = 1 reproduces the reference (which has no scaling, and one head).
 * Small graphs run each window on a team of 4 or 16 waves of one workgroup
 * (masked: W*H <= 1024, teams of 4; tile-dense: W*H <= 512, teams of 16, up
 * to 2048, teams of 4), each wave taking an even share of the window's
 * tiles, merged in LDS in a fixed order, in the order's sequence.  On larger
 * graphs (W > 512), given d_window_order on a launch of fewer than 2^18
 * window-heads (W x H), windows run in the order's sequence: the heavy
 * windows (more than max(1024, 8 x mean) tiles) among its first 512 entries
 * as teams of 4 waves in the launch's first workgroups, every other entry on
 * one wave.  In natural order, and with an order from 2^18 window-heads on,
 * the order only names the windows -- each named window is computed once;
 * invalid entries are skipped -- and the library schedules them itself,
 * identically for every order: the heavy windows, heaviest first, the first
 * W / 8 / H of them (64 to 512) as such teams; every other window on one
 * wave, by octave of its tile count, heaviest first, each octave in index
 * order and cut into eight contiguous shares interleaved slot by slot across
 * the XCDs (longest windows first for the tail, each share's contiguous
 * windows on one or a few XCDs for the L2; on a community-ordered graph the
 * reference's descending order would scatter each community over the whole
 * run).  Either way, where the heaviest window would outlast the rest of the
 * pass on four waves (by T x H and, masked, its attended columns), the first
 * up to 64 heavy entries run as teams of 16 waves in a launch before it.
 * With W <= 1024 no window can be heavy (one tile per block column at most)
 * and no teams are launched.  Three small kernels (four given an order;
 * ~15-30 us; one for the three up to 4,096 windows) build the schedule in
 * scratch of about 9 bytes per window taken from the library's cache and
 * returned to it in stream order on `stream` (the call
 * does not wait).  Tensors past ~4 GiB take the sequence of the order, as
 * small graphs do.  Every other path allocates nothing. */
f3s_status f3s_attention_fwd(const uint16_t* Q, const uint16_t* K, const uint16_t* V,
                             float* O, const int32_t* d_window_offsets,
                             const int32_t* d_block_col, const uint16_t* d_tile_mask,
                             const int32_t* d_window_order, int32_t W, int32_t n,
                             int32_t d, int32_t H, float scale, void* stream);

/* f3s_attention_fwd without any device allocation.  No counterpart in the
 * reference: for callers that cannot allocate (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc).  Same arguments,
 * semantics, kernels and results (bit for bit) as f3s_attention_fwd; the
 * schedule's scratch (tables, team list, class counts, one-wave slots and an
 * order's inverse: 16.5 MiB) is a fixed device array of the library, one per
 * GPU, held until the process ends.  Limit: W <= 2,097,152 row windows
 * (n <= 33,554,432 nodes); larger W returns F3S_EUNSUPPORTED.  Every call on
 * one GPU shares that GPU's array and overwrites it, so calls that overlap in
 * time on one GPU (e.g. on two streams) race; serialise them.  Allocates
 * nothing, clears no memory and never waits for the device. */
f3s_status f3s_attention_fwd_noalloc(const uint16_t* Q, const uint16_t* K, const uint16_t* V,
                                     float* O, const int32_t* d_window_offsets,
                                     const int32_t* d_block_col, const uint16_t* d_tile_mask,
                                     const int32_t* d_window_order, int32_t W, int32_t n,
                                     int32_t d, int32_t H, float scale, void* stream);

/* The timed launch of tests/test_fused_3s_v2.cu:126-136 (events recorded
 * around the kernel on the launch stream): `reps` back-to-back calls of
 * f3s_attention_fwd with the same arguments, timed with HIP events on
 * `stream`; *us_out = mean microseconds per call.  Synchronises `stream`. */
f3s_status f3s_attention_fwd_timed(const uint16_t* Q, const uint16_t* K, const uint16_t* V,
                                   float* O, const int32_t* d_window_offsets,
                                   const int32_t* d_block_col, const uint16_t* d_tile_mask,
                                   const int32_t* d_window_order, int32_t W, int32_t n,
                                   int32_t d, int32_t H, float scale, void* stream,
                                   int32_t reps, float* us_out);

/* f3s_naive_baseline_kernel (baselines/gpu_baseline.cu:28-116): the naive
 * edge-exact comparator, one thread per node, fp32 Q/K/V/O [n][d], CSR
 * neighbours as stored (a duplicate entry counts twice, as in
 * cpu_sparse_attention_csr).  No device-heap allocation (the reference
 * mallocs per thread).  1 <= d <= 64. */
f3s_status f3s_naive_attention_fwd(const float* Q, const float* K, const float* V, float* O,
                                   const int32_t* d_row_ptr, const int32_t* d_col_idx,
                                   int32_t n, int32_t d, float scale, void* stream);

/* Planned execution (no reference counterpart; the reference relies on the
 * window sort alone, include/utils.cuh:48-59).  A plan splits windows with
 * more than `seg_tiles` tiles into segments processed by separate waves; the
 * last segment of each split window to finish merges its segments in a fixed
 * order (deterministic), inside the same launch, so hub windows do not
 * serialise.  seg_tiles = 0 chooses
 * automatically: on small graphs (W*H <= 2048) the teams of f3s_attention_fwd
 * (same items, same bits), else segment sizes from T*H.  Windows run in d_window_order (the reference's descending
 * sort) or, when it is NULL, in natural order with consecutive windows kept
 * on one XCD (for community-ordered graphs).  Build once per graph; reuse for
 * every forward pass; one plan must not serve two overlapping calls (it owns
 * the partial-result buffers).  From 2^18 window-heads (W x H) on, a plan
 * whose items run one wave each follows the library's schedule of
 * f3s_attention_fwd instead of the order's sequence (the order then only
 * names the windows), keeping a community-ordered graph's L2 reuse under the
 * reference's descending order. */
typedef struct f3s_plan f3s_plan;
f3s_status f3s_plan_create(const int32_t* d_window_offsets, const int32_t* d_window_order,
                           int32_t W, int32_t H, int32_t seg_tiles, void* stream,
                           f3s_plan** plan_out);
/* f3s_plan_create (automatic segments) whose items follow the library's
 * schedule from 513 windows on, wherever masked passes run no teams (past 1,024
 * window-heads), not only from 2^18 window-heads: each class's windows in eight
 * contiguous shares, one for each XCD.  Fewer windows keep their natural order.
 * For passes of longer rows, which gain more from a community-ordered graph's
 * L2 reuse (f3s_diff_attention_fwd). */
f3s_status f3s_plan_create_scheduled(const int32_t* d_window_offsets, int32_t W, int32_t H,
                                     void* stream, f3s_plan** plan_out);
f3s_status f3s_plan_destroy(f3s_plan* plan);
/* Lists, once per graph, the columns each planned item attends under the
 * masked semantics (32 row offsets + 32 row masks per 32-column chunk), so
 * masked passes read 8 bytes per attended column instead of expanding 36
 * bytes of tile metadata on every pass.  Later masked calls of
 * f3s_attention_fwd_planned with these same d_block_col / d_tile_mask
 * pointers and n use the lists; the structure they point to must not change
 * afterwards (compile again if it does).  Other calls are unaffected. */
f3s_status f3s_plan_compile(f3s_plan* plan, const int32_t* d_block_col,
                            const uint16_t* d_tile_mask, int32_t n, void* stream);
f3s_status f3s_plan_info(const f3s_plan* plan, int64_t* num_items, int64_t* num_split_windows,
                         int64_t* T, int32_t* seg_tiles);
/* The sizes behind a planned pass's memory traffic (no reference
 * counterpart): compiled column chunks (256 bytes each; 0 before
 * f3s_plan_compile), and for the item sets of masked and of tile-dense
 * passes their work items (16 bytes each) and split-window partial slots
 * (per head, 4,224 bytes written by the pass and read by its merge).  Any
 * output pointer may be NULL. */
f3s_status f3s_plan_stats(const f3s_plan* plan, int64_t* num_chunks, int64_t* masked_items,
                          int64_t* masked_slots, int64_t* dense_items, int64_t* dense_slots);
f3s_status f3s_attention_fwd_planned(const f3s_plan* plan, const uint16_t* Q,
                                     const uint16_t* K, const uint16_t* V, float* O,
                                     const int32_t* d_block_col, const uint16_t* d_tile_mask,
                                     int32_t n, int32_t d, int32_t H, float scale,
                                     void* stream);

/* The masked pass of a compiled plan on one packed tensor QKV [n][3][H][64]
 * (what a single projection of the node features writes: Q, K and V are its
 * thirds) with O [n][H][64] in float32 or, with out_half, in binary16 (the
 * float32 result rounded once, to nearest even).  No reference counterpart:
 * a layer needs no copies of Q, K and V and no cast of O around the pass.
 * Same results, bit for bit, as f3s_attention_fwd_planned on the copies.
 * F3S_EINVAL unless the plan was compiled for this n; F3S_EUNSUPPORTED past
 * n * H * 384 bytes = 4 GiB less 48 KiB. */
f3s_status f3s_attention_fwd_packed(const f3s_plan* plan, const uint16_t* QKV, void* O,
                                    int32_t out_half, int32_t n, int32_t d, int32_t H,
                                    float scale, void* stream);

/* The projections around the fused pass (no reference counterpart): Y[n][M] =
 * X[n][K] W[M][K]^T + bias[M] (NULL: none), all binary16, sums in float32,
 * rounded once.  K a multiple of 8 up to 256, M a multiple of 32 up to 32768,
 * X, W and Y 16-byte aligned; F3S_EUNSUPPORTED otherwise.  Asynchronous on
 * `stream`. */
f3s_status f3s_linear_f16(const uint16_t* X, const uint16_t* W, const uint16_t* bias, uint16_t* Y,
                          int64_t n, int32_t K, int32_t M, void* stream);

/* A projection with its epilogue (no reference counterpart), of any size:
 *   Y[n][M] = act(X[n][K] W[M][K]^T + bias[M]) + R[n][M]
 * in `dtype` (F3S_F16 or F3S_BF16), sums and epilogue in float32, rounded once.
 * bias and R may be NULL.  Rows of X and R are x_stride and r_stride values
 * apart; W and Y are contiguous.  No alignment is needed; rows of a multiple of
 * 16 bytes at 16-byte addresses are the fast ones.  K, M < 2^22, n < 2^36.
 * workspace: f3s_linear_workspace bytes, 16-byte aligned, this call's alone
 * until it is done; nothing is allocated, calls may overlap and be captured.
 * Deterministic.  Asynchronous on `stream`. */
#define F3S_ACT_NONE 0
#define F3S_ACT_RELU 1
#define F3S_ACT_GELU 2        /* z Phi(z) */
#define F3S_ACT_GELU_TANH 3   /* its tanh approximation */
#define F3S_ACT_SILU 4
f3s_status f3s_linear_workspace(int64_t n, int64_t K, int64_t M, int32_t act, int32_t backward_pass,
                                int64_t* bytes);
/* How a product of such a call runs, for tests and measurements: F3S_LINEAR_FORWARD, the
 * backward pass's SLOPE (z again; with an activation), DX or DW (`bias`: with db), of
 * contiguous 16-byte-aligned tensors.  kernel: up to 64 rows, W held in LDS, or tiles;
 * tiles only: their side, splits of the contraction, tiles and workgroups of each split
 * (fewer workgroups take several tiles each); pieces: 2 whole 16-byte pieces everywhere,
 * 1 in the operands' rows, 0 neither.  Any output may be NULL. */
#define F3S_LINEAR_FORWARD 0
#define F3S_LINEAR_SLOPE 1
#define F3S_LINEAR_DX 2
#define F3S_LINEAR_DW 3
#define F3S_LINEAR_FEW_ROWS 0
#define F3S_LINEAR_W_IN_LDS 1
#define F3S_LINEAR_TILES 2
f3s_status f3s_linear_tiling(int64_t n, int64_t K, int64_t M, int32_t act, int32_t bias,
                             int32_t product, int32_t* kernel, int32_t* tile, int32_t* splits,
                             int64_t* tiles, int64_t* workgroups, int32_t* pieces);
f3s_status f3s_linear_fwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                          const uint16_t* bias, const uint16_t* R, int64_t r_stride, uint16_t* Y,
                          int64_t n, int64_t K, int64_t M, int32_t act, int32_t dtype,
                          void* workspace, int64_t workspace_bytes, void* stream);
/* Its gradient: dX[n][K], dW[M][K], db[M] (contiguous; NULL: not wanted) from
 * dY, whose rows are dy_stride values apart (dR is dY).  With an activation z is
 * computed again from X, W and bias: the forward call keeps nothing.  Sums are
 * float32.  dZ = dY act'(Z) is rounded to `dtype` before dX = dZ W and dW = dZ^T X
 * are made of it, so these two carry its rounding and their own; db is summed
 * before that.  Without an activation dZ is dY: one rounding each. */
f3s_status f3s_linear_bwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                          const uint16_t* bias, const uint16_t* dY, int64_t dy_stride, uint16_t* dX,
                          uint16_t* dW, uint16_t* db, int64_t n, int64_t K, int64_t M, int32_t act,
                          int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream);

/* The reversed edges of a CSR (no reference counterpart): entry (i, j) becomes
 * (j, i).  d_out_row_ptr holds n + 1 entries, d_out_col_idx nnz.  The order of
 * the entries of a row is not defined (the converter's output does not depend on
 * it).  Columns outside [0, n) are left out, and the converter then refuses the
 * result.  Asynchronous on `stream`; scratch from the library's cache. */
f3s_status f3s_reverse_csr(const int32_t* d_row_ptr, const int32_t* d_col_idx, int32_t n,
                           int64_t nnz, int32_t* d_out_row_ptr, int32_t* d_out_col_idx,
                           void* stream);

/* Differential attention over the edges of a compiled plan (no reference
 * counterpart): per head two maps of 64 dims, q = [q1 q2], k = [k1 k2], and
 * values of 128,
 *   O[i] = sum_j (softmax_j(scale q1.k1) - lam[h] softmax_j(scale q2.k2)) V[j]
 * over the edges (i, j) (masked semantics); rows without edges get 0.  H is the
 * plan's; a head of a row is 128 contiguous values of `dtype` (F3S_F16 or
 * F3S_BF16), heads adjacent, rows `*_stride` values apart (a multiple of 8, at
 * least H * 128), pointers 16-byte aligned: the thirds of a packed
 * [n][3][H][128] tensor are taken as they lie.  lam float32 [H].  lse, where
 * not NULL, receives [n][H][2] float32 for the gradient.  Sums and softmax
 * statistics are float32, O is rounded once.  An infinite or NaN value reaches
 * the rows with an edge to its node only (an infinite value of V makes their
 * sums NaN).  A row whose logits are all -inf is 0 if both maps' are, as one
 * without edges, else NaN.  Logits past 2^26 in size may come out as NaN: float32
 * holds them to whole units only.  Deterministic.
 * workspace: f3s_diff_attention_workspace bytes (reversed NULL), 16-byte
 * aligned, this call's alone until it is done; nothing else is allocated or
 * kept, so calls may overlap and be captured.  Asynchronous on `stream`. */
f3s_status f3s_diff_attention_workspace(const f3s_plan* plan, const f3s_plan* reversed,
                                        int64_t* bytes);
f3s_status f3s_diff_attention_fwd(const f3s_plan* plan, const uint16_t* Q, int64_t q_stride,
                                  const uint16_t* K, int64_t k_stride, const uint16_t* V,
                                  int64_t v_stride, const float* lam, uint16_t* O, int64_t o_stride,
                                  float* lse, int32_t dtype, int32_t n, int32_t H, float scale,
                                  void* workspace, int64_t workspace_bytes, void* stream);
/* Its gradient: dQ, dK, dV in `dtype`, dlam float32 [H], from dO and the
 * forward call's lse.  `reversed` is a plan of the reversed edges
 * (f3s_reverse_csr, converted) of the same n and H, compiled.  No atomics:
 * deterministic.  F3S_EUNSUPPORTED from n * H = 2^28 on. */
f3s_status f3s_diff_attention_bwd(const f3s_plan* plan, const f3s_plan* reversed,
                                  const uint16_t* Q, int64_t q_stride, const uint16_t* K,
                                  int64_t k_stride, const uint16_t* V, int64_t v_stride,
                                  const float* lam, const float* lse, const uint16_t* dO,
                                  int64_t do_stride, uint16_t* dQ, int64_t dq_stride, uint16_t* dK,
                                  int64_t dk_stride, uint16_t* dV, int64_t dv_stride, float* dlam,
                                  int32_t dtype, int32_t n, int32_t H, float scale, void* workspace,
                                  int64_t workspace_bytes, void* stream);

/* Measurement only (no reference counterpart): the device's random-gather
 * ceiling for the fused pass's access pattern.  For each of `count` columns
 * (a multiple of 32) it loads the 128-byte row at byte offset
 * d_idx[i] * row_stride of K and of V (eight lanes x 16 bytes per row, 32
 * columns per step, `cpw` steps per wave: the fused pass's load shape) and
 * folds the bytes into d_out, one word per wave: ceil(count / 32 / cpw)
 * words.  Tables hold `rows` rows (rows * row_stride <= 0xffff0000 bytes);
 * a negative row or one past the table reads zero.  Asynchronous on
 * `stream`. */
f3s_status f3s_probe_gather(const uint16_t* K, const uint16_t* V, int64_t rows,
                            int32_t row_stride, const int32_t* d_idx, int64_t count,
                            int32_t cpw, uint32_t* d_out, void* stream);

#ifdef __cplusplus
}
#endif
#endif
