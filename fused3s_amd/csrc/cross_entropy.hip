// cross_entropy.hip -- the cross entropy of a linear classifier over many classes, and
// its gradient, without keeping the logits, binary16 and bfloat16.
//
//   z = x W^T + b,  loss_i = log sum_c exp z_ic - z_it,  t the row's target
//   dz_ic = g_i (exp(z_ic) / sum - [c = t]),  g the loss's gradient (mean: over the
//   number of rows that count),  dx = dz W,  dW = dz^T x,  db = sum_i dz
//
// The products are the tiled ones of projections (gemm_tiles.hpp):
//   forward  z in the registers of a tile; its epilogue leaves, for each row and block
//            of 32 or 64 classes, the largest z and the sum of exp(z - that), 8 bytes,
//            and z at the target; a second launch joins a row's blocks
//   backward in pieces of the classes: z again, dz of a piece in its epilogue, in the
//            type, then its share of dx (float32, added up over the pieces) and its
//            rows of dW.  A piece's dz is kPieceBytes at most: past kPieceRows rows they
//            are taken a block at a time, and dW is added up over the blocks (float32).
//            So memory goes with V K and a block's K, not with n V, for one product of
//            four more than keeping z would take.
// Of few inputs (K <= 256) the logits, and dz, stay in registers: below.
// dz is rounded to the type, the operand that dx and dW take: these two carry that
// rounding beside their own; db is summed before it.  (Of few classes, where bytes bound
// the passes and not products, it goes on as the sum of two 16-bit values.)  What dz is multiplied with
// throughout (1 / count, a loss scale) comes last, in float32, so that small gradients
// do not vanish: dz itself is of size 1 at most, in binary16 times 2^14, as a class
// of probability 4e-9 still has its 11 bits then.  (As two 16-bit values it would take a
// product more for each of dx and dW: with few inputs 52,802 x 64 -> 10,778 trained 675 ->
// 821 us, 16,384 x 256 -> 50,021 2,264 -> 2,679; where dz goes through memory twice its
// bytes too.  Rounded, these gradients are at most 1.41 times as far off as by their own
// rounding alone.)
// What bounds it is the matrix cores, with many classes; with few, x.
#include <cmath>

#include "gemm_tiles.hpp"

namespace f3s {

// (16,384 x 512 -> 100,003, a training step, milliseconds with pieces of 128, 256, 512 and
// 1,024 MB: 8.9, 8.9, 8.5, 9.1: fewer launches and additions of dx against what the
// Infinity Cache holds.)
constexpr int64_t kPieceBytes = 512 << 20;    // of dz
constexpr int64_t kPieceRows = kPieceBytes / 2 / 1024;   // so that a piece has 1,024 classes
constexpr int64_t kBlocksBytes = 256 << 20;   // of a forward pass's blocks
constexpr int kLossThreads = 256;

enum Reduction : int { kNone = 0, kMean = 1, kSum = 2 };

struct CeParams {
    const int64_t* target;
    int64_t n, V, ignore;
    const float2* blocks;    // [nblocks][rows]
    int64_t nblocks, rows, first_row;
    const float* picked;     // [rows]
    float* lse;              // [n + 1]; last: the rows that count (NULL: not)
    float* loss;             // [n] or [1]
    double* parts;           // [workgroups][2]: loss, count
    int64_t nparts;
    int32_t reduction;
};

// A row's blocks joined: ROWS rows by the other threads' parts of the blocks, in a fixed
// order.  (64 rows of 1,564 blocks, 16 rows a workgroup: 16 us, four: 8; 200,003 rows of
// two blocks, 16: 15, 256: 5.)
template <int ROWS>
__global__ void __launch_bounds__(kLossThreads) loss_join(const CeParams p)
{
    constexpr int kParts = kLossThreads / ROWS;
    __shared__ float2 lds[kParts][ROWS + 1];
    const int in = threadIdx.x % ROWS, part = threadIdx.x / ROWS;
    const int64_t row = (int64_t)blockIdx.x * ROWS + in, i = p.first_row + row;
    const int64_t per = (p.nblocks + kParts - 1) / kParts, first = part * per,
                  end = min(p.nblocks, first + per);
    float m = -INFINITY, s = 0.f;
    auto take = [&](float2 b) {
        // (a NaN block's largest may not be NaN, its sum is)
        const float top = __builtin_fmaxf(m, b.x);
        const float mu = top == -INFINITY ? 0.f : top;
        s = s * fast_exp2((m - mu) * 1.44269504f) + b.y * fast_exp2((b.x - mu) * 1.44269504f);
        m = top;
    };
    if (row < p.rows)
        for (int64_t k = first; k < end; k += 8) {
            float2 b[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) b[u] = p.blocks[min(k + u, end - 1) * p.rows + row];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k + u < end) take(b[u]);
        }
#pragma unroll
    for (int step = kParts / 2; step >= 1; step /= 2) {   // part k takes k + step
        if (part >= step && part < 2 * step) lds[part][in] = make_float2(m, s);
        __syncthreads();
        if (part < step) take(lds[part + step][in]);
    }
    double loss = 0.0, counts = 0.0;
    if (part == 0) {
        if (row < p.rows) {
            const int64_t t = p.target[i];
            const bool none = t == p.ignore;
            const float l = 0.69314718f * __log2f(s);
            float value = 0.f;
            if (!none)   // (a target that is no class: NaN)
                value = t < 0 || t >= p.V ? NAN : (m - p.picked[row]) + l;
            if (p.lse) p.lse[i] = m + l;
            if (p.reduction == kNone) p.loss[i] = value;
            loss = value;
            counts = none ? 0.0 : 1.0;
        }
    }
    __shared__ double sums[kLossThreads / kWave][2];
    loss = wave_sum(loss);
    counts = wave_sum(counts);
    if (threadIdx.x % kWave == 0) {
        sums[threadIdx.x / kWave][0] = loss;
        sums[threadIdx.x / kWave][1] = counts;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        double t = 0.0;
        for (int k = 0; k < kLossThreads / kWave; ++k) t += sums[k][threadIdx.x];
        p.parts[2 * (p.first_row / ROWS + blockIdx.x) + threadIdx.x] = t;
    }
}

// The workgroups' sums in order.
__global__ void __launch_bounds__(1024) loss_total(const CeParams p)
{
    __shared__ double lds[2][1024 / kWave];
    double s[2] = {0.0, 0.0};
    for (int64_t k = threadIdx.x; k < p.nparts; k += 8 * 1024) {
        double2 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            x[u] = reinterpret_cast<const double2*>(p.parts)[min(k + u * 1024, p.nparts - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (k + u * 1024 < p.nparts) {
                s[0] += x[u].x;
                s[1] += x[u].y;
            }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        s[c] = wave_sum(s[c]);
        if (threadIdx.x % kWave == 0) lds[c][threadIdx.x / kWave] = s[c];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double loss = 0.0, count = 0.0;
        for (int k = 0; k < 1024 / kWave; ++k) {
            loss += lds[0][k];
            count += lds[1][k];
        }
        if (p.reduction == kMean) p.loss[0] = (float)(loss / count);   // (no row counts: NaN)
        if (p.reduction == kSum) p.loss[0] = (float)loss;
        if (p.lse) p.lse[p.n] = (float)count;
    }
}

// ---- what multiplies dz: row i's f, and the factor of the results ----

// The largest |dloss| of blockIdx.x's share (reduction none, binary16).
__global__ void __launch_bounds__(kLossThreads)
loss_largest(const float* __restrict__ dloss, int64_t n, float* __restrict__ parts)
{
    __shared__ float lds[kLossThreads / kWave];
    float m = 0.f;
    for (int64_t i = (int64_t)blockIdx.x * kLossThreads + threadIdx.x; i < n;
         i += (int64_t)gridDim.x * kLossThreads) {
        const float x = __builtin_fabsf(dloss[i]);
        m = x <= 3.4e38f ? __builtin_fmaxf(m, x) : m;   // (infinite and NaN: their own rows')
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, off, kWave));
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kLossThreads / kWave; ++k) m = __builtin_fmaxf(m, lds[k]);
        parts[blockIdx.x] = m;
    }
}

struct FactorParams {
    const int64_t* target;
    int64_t n, V, ignore;
    const float* dloss;
    const float* count;
    const float* largest;   // [many] or NULL
    int32_t many, reduction;
    float lift;
    float* f;               // [n]
    float* factor;
};
__global__ void __launch_bounds__(kLossThreads) loss_factors(const FactorParams p)
{
    float unit = 1.f;   // a power of two
    if (p.largest) {
        float m = 0.f;
        for (int k = 0; k < p.many; ++k) m = __builtin_fmaxf(m, p.largest[k]);
        // (kept where it over 2^14 and that's inverse are ones too)
        const int e = m > 0.f ? __builtin_amdgcn_frexp_expf(m) : 0;
        unit = __builtin_amdgcn_ldexpf(1.f, e < -110 ? -110 : e > 120 ? 120 : e);
    }
    const int64_t i = (int64_t)blockIdx.x * kLossThreads + threadIdx.x;
    if (i < p.n) {
        const int64_t t = p.target[i];
        p.f[i] = t == p.ignore           ? 0.f
                 : t < 0 || t >= p.V     ? NAN
                 : p.reduction == kNone  ? p.dloss[i] * (p.lift / unit)
                                         : p.lift;
    }
    if (i == 0)
        *p.factor = (p.reduction == kNone ? unit : p.dloss[0]) / p.lift /
                    (p.reduction == kMean ? __builtin_fmaxf(*p.count, 1.f) : 1.f);   // (0: all dz are)
}

// Slices of a product added, times the factor.
template <typename T>
__global__ void __launch_bounds__(256)
join_scaled(const float* __restrict__ parts, int64_t count, int32_t slices,
            const float* __restrict__ factor, T* __restrict__ out)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = (T)(split_sum(parts + i, count, 0, slices) * *factor);
}
// Slices of one of several blocks' product added onto those of the blocks before; after
// the last block, times the factor.
template <typename T>
__global__ void __launch_bounds__(256)
join_blocks(const float* __restrict__ parts, int64_t count, int32_t slices, float* __restrict__ sums,
            bool first, bool last, const float* __restrict__ factor, T* __restrict__ out)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const float s = (first ? 0.f : sums[i]) + split_sum(parts + i, count, 0, slices);
        if (last) out[i] = (T)(s * *factor);
        else sums[i] = s;
    }
}
template <typename T>
__global__ void __launch_bounds__(256)
cast_scaled(const float* __restrict__ in, int64_t count, const float* __restrict__ factor,
            T* __restrict__ out)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) out[i] = (T)(in[i] * *factor);
}

template <typename T>
__global__ void __launch_bounds__(256) loss_zero(T* __restrict__ out, int64_t count)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = (T)0.f;
}

// ---- log-sum-exps of few inputs: K <= 256, whole pieces ----
//
// There a tile's products are short beside its epilogue, which nothing overlaps.  So a
// wave keeps 32 rows of x in registers and the classes stream past it, 64 at a time,
// through LDS, the next ones on their way; several workgroups share a CU.  A lane keeps
// the largest logit and the sum of its own classes: nothing crosses lanes before the
// end, and a row leaves one block for each share of the classes (blockIdx.y), not one
// for each 64.  Bound by the logits' 8 operations each, one exponential among them.
// (A logit is taken from the largest before log2(e): z log2(e) - m log2(e) in one
// operation less rounds, or overflows, what should be 0: at logits of 1,000 losses were
// 3e-5 below 0.  52,802 x 64 -> 10,778 143 us so, 153 as it is; x 128 the same.)
// (By tiles and so, us a call: 52,802 x 64 -> 10,778 411 and 153;
// 200,003 x 128 -> 300 70 and 41; 16,384 x 256 -> 50,021 743 and 430.)
constexpr int kStreamWaves = 4, kStreamTiles = 2, kStreamRows = 16 * kStreamTiles * kStreamWaves;
struct StreamParams {
    const char *x, *w, *bias;
    int64_t ldx, rows, V;
    int32_t K;
    int64_t per;             // chunks of 64 classes in a share
    const int64_t* target;
    float2* blocks;          // [shares][rows]
    float* picked;           // [rows]
};
template <typename T, int KS>
__global__ void __launch_bounds__(kStreamWaves * kWave) stream_lse_kernel(const StreamParams p)
{
    typedef typename Half<T>::v8 v8;
    constexpr int kChunkBytes = 64 * kStep * 2;   // 64 classes by 64 inputs
    __shared__ __align__(256) char wl[2][KS * kChunkBytes];
    __shared__ __align__(16) float bl[2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int64_t first = (int64_t)blockIdx.x * kStreamRows + wave * 16 * kStreamTiles;
    const int64_t chunks = (p.V + 63) / 64, begin = blockIdx.y * p.per,
                  end = min(chunks, begin + p.per);
    typedef TileAt<false, 64, kStreamWaves> At;
    float next_bias = 0.f;
    auto load = [&](int64_t c, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
            load_tile(At(p.w, p.K, 64 * c, p.V, kStep * k, p.K), p.K, wl[buf] + k * kChunkBytes, wave,
                      lane);
        const int64_t at = 64 * c + threadIdx.x;
        if (threadIdx.x < 64)
            next_bias = at >= p.V ? -INFINITY
                        : p.bias  ? (float)reinterpret_cast<const T*>(p.bias)[at]
                                  : 0.f;
    };
    if (begin < end) load(begin, 0);
    v8 x[kStreamTiles][2 * KS];
    int64_t t[kStreamTiles];
    float m[kStreamTiles], s[kStreamTiles];
#pragma unroll
    for (int u = 0; u < kStreamTiles; ++u) {
        const int64_t row = min(first + 16 * u + r, p.rows - 1);
        const T* src = reinterpret_cast<const T*>(p.x) + row * p.ldx + 8 * g;
        t[u] = p.target[row];
        m[u] = -INFINITY;
        s[u] = 0.f;
#pragma unroll
        for (int f = 0; f < 2 * KS; ++f) {
            x[u][f] = v8{};
            if (32 * f + 8 * g < p.K) x[u][f] = *reinterpret_cast<const v8*>(src + 32 * f);
        }
    }
    int buf = 0;
    for (int64_t c = begin; c < end; ++c, buf ^= 1) {
        // (loads into LDS are waited for by hand: the barrier does not)
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        if (threadIdx.x < 64) bl[buf][threadIdx.x] = next_bias;
        __syncthreads();
        if (c + 1 < end) load(c + 1, buf ^ 1);
        f4 z[4][kStreamTiles];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < kStreamTiles; ++u)
                z[i][u] = *reinterpret_cast<const f4*>(&bl[buf][16 * i + 4 * g]);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v8 a = fragment<T, false, 64>(wl[buf] + k * kChunkBytes, i, f, lane);
#pragma unroll
                    for (int u = 0; u < kStreamTiles; ++u)
                        z[i][u] = Half<T>::mfma(a, x[u][2 * k + f], z[i][u]);
                }
#pragma unroll
        for (int u = 0; u < kStreamTiles; ++u) {
            float top = m[u];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) top = __builtin_fmaxf(top, z[i][u][v]);
            const float mu = top == -INFINITY ? 0.f : top;
            float sum = s[u] * fast_exp2((m[u] - mu) * kLog2eF);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) sum += fast_exp2((z[i][u][v] - mu) * kLog2eF);
            s[u] = sum;
            m[u] = top;
            const int64_t at = t[u] - 64 * c;
            if (__ballot(at >= 0 && at < 64)) {
                float picked = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) picked = at == 16 * i + 4 * g + v ? z[i][u][v] : picked;
                const int64_t row = first + 16 * u + r;
                if (at >= 0 && at < 64 && t[u] < p.V && ((at >> 2) & 3) == g && row < p.rows)
                    p.picked[row] = picked;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kStreamTiles; ++u) {
        const float top = row_max4(m[u]);
        float sum = s[u] * fast_exp2((m[u] - (top == -INFINITY ? 0.f : top)) * kLog2eF);
        sum += __shfl_xor(sum, 16, kWave);
        sum += __shfl_xor(sum, 32, kWave);
        const int64_t row = first + 16 * u + r;
        if (g == 0 && row < p.rows)
            p.blocks[(int64_t)blockIdx.y * p.rows + row] = make_float2(top, sum);
    }
}

// ---- their gradients: K <= 256, whole pieces ----
//
// dz never leaves the registers: two passes of one shape, each with the logits again.
// A wave keeps 32 rows of its own (16 past 128 inputs, whose sums fill the registers),
// the others stream past it, 64 at a time:
//   dx      its rows are x's, W's stream past: dx += dz W
//   dW, db  its rows are W's, x's stream past: dW += dz^T x
// A lane's logits of a row are the operand of the product after them, whose other one is
// the same rows in LDS, read transposed.  Shares of the streamed rows (blockIdx.y) are
// added by join_scaled.  One product of five more than by tiles, and none of dz's bytes.
// (A training step by tiles and so, us: 52,802 x 64 -> 10,778 1,324 and 672; x 128 1,473
// and 879; x 256 2,147 and 1,669; 16,384 x 256 -> 50,021 3,277 and 2,303.)
struct GradParams {
    const char *own, *other;
    int64_t ld_own, ld_other, owns, others;
    int32_t K;
    int64_t per;             // chunks of 64 of the others in a share
    const char* bias;
    const int64_t* target;   // of x's rows
    const float *lse, *f;
    const float* factor;
    char* out;               // [owns][K] in the type, times the factor: one share; else
    float* slices;           // [shares][owns][K]
    float* sums;             // db: [shares][owns] (NULL: not wanted)
};
__device__ __forceinline__ int place_both(int row) { return (row & 6) | ((row >> 3) & 1); }
template <typename T, int KS, int TILES, bool CLASSES>
__global__ void __launch_bounds__(kStreamWaves * kWave) __attribute__((amdgpu_waves_per_eu(2)))
stream_grad_kernel(const GradParams p)
{
    typedef typename Half<T>::v8 v8;
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* lds4;
    constexpr int kRows = 16 * TILES * kStreamWaves;   // of its own
    constexpr int kBytes = 64 * kStep * 2, kDims = 4 * KS;   // 64 rows by 64 inputs; tiles of dims
    __shared__ __align__(256) char rows[2][KS * kBytes];
    __shared__ __align__(16) float at1[2][64], at2[2][64];    // bias; lse and f
    __shared__ __align__(16) int32_t at3[2][64];              // (CLASSES) targets, of the wave's classes
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int64_t block0 = (int64_t)blockIdx.x * kRows, first = block0 + wave * 16 * TILES;
    const int64_t chunks = (p.others + 63) / 64, begin = blockIdx.y * p.per,
                  end = min(chunks, begin + p.per);
    float next1 = 0.f, next2 = 0.f;
    int32_t next3 = -1;
    auto load = [&](int64_t c, int buf) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs =
            make_rsrc(p.other + 64 * c * p.ld_other * 2, 0x7fffffffu);
        const int64_t left = p.others - 64 * c;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {   // 1,024 bytes a wave and load, eight rows
                const int part = i * kStreamWaves + wave, row = part * 8 + lane / 8;
                const int piece = (lane % 8) ^ place_both(row);
                const bool in = row < left && kStep * k + 8 * piece < p.K;
                const uint32_t at =
                    in ? (uint32_t)(row * (int32_t)p.ld_other + kStep * k + 8 * piece) * 2 : 0xffffff00u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rs, (__attribute__((address_space(3))) void*)(rows[buf] + k * kBytes + part * 1024),
                    16, (int)at, 0, 0, 0);
            }
        const int64_t at = 64 * c + threadIdx.x;
        if (threadIdx.x < 64) {
            if constexpr (CLASSES) {
                const bool in = at < p.others;
                next1 = in ? p.lse[at] : 0.f;
                next2 = in ? p.f[at] : 0.f;
                const int64_t t = in ? p.target[at] - block0 : -1;
                next3 = t >= 0 && t < kRows ? (int32_t)t : -1;
            } else {
                next1 = at >= p.others ? -INFINITY
                        : p.bias       ? (float)reinterpret_cast<const T*>(p.bias)[at]
                                       : 0.f;
            }
        }
    };
    if (begin < end) load(begin, 0);
    v8 own[TILES][2 * KS];
    float own1[TILES], own2[TILES], sum[TILES];   // lse, f; bias
    int64_t t[TILES];
    f4 acc[TILES][kDims];
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
        const int64_t row = min(first + 16 * u + r, p.owns - 1);
        const T* src = reinterpret_cast<const T*>(p.own) + row * p.ld_own + 8 * g;
#pragma unroll
        for (int f = 0; f < 2 * KS; ++f) {
            own[u][f] = v8{};
            if (32 * f + 8 * g < p.K) own[u][f] = *reinterpret_cast<const v8*>(src + 32 * f);
        }
        if constexpr (CLASSES) {
            own1[u] = p.bias ? (float)reinterpret_cast<const T*>(p.bias)[row] : 0.f;
        } else {
            own1[u] = p.lse[row];
            own2[u] = p.f[row];
            t[u] = p.target[row];
        }
        sum[u] = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[u][d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    int buf = 0;
    for (int64_t c = begin; c < end; ++c, buf ^= 1) {
        // (loads into LDS are waited for by hand: the barrier does not)
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        if (threadIdx.x < 64) {
            at1[buf][threadIdx.x] = next1;
            if constexpr (CLASSES) {
                at2[buf][threadIdx.x] = next2;
                at3[buf][threadIdx.x] = next3;
            }
        }
        __syncthreads();
        if (c + 1 < end) load(c + 1, buf ^ 1);
        // logits of the chunk's rows 16 i + 4 g + v and own row r
        f4 z[4][TILES];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < TILES; ++u)
                z[i][u] = CLASSES ? f4{own1[u], own1[u], own1[u], own1[u]}
                                  : *reinterpret_cast<const f4*>(&at1[buf][16 * i + 4 * g]);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v8 a = *reinterpret_cast<const v8*>(
                        rows[buf] + k * kBytes + (16 * i + r) * 128 +
                        16 * ((4 * f + g) ^ place_both(r)));
#pragma unroll
                    for (int u = 0; u < TILES; ++u)
                        z[i][u] = Half<T>::mfma(a, own[u][2 * k + f], z[i][u]);
                }
        // dz in their place
        uint64_t hits = 0;   // (CLASSES) whether a target is among the wave's classes
        if constexpr (CLASSES) {
            const int32_t at = at3[buf][lane];
            hits = __ballot(at >= 0 && at / (16 * TILES) == wave);
        }
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f4 lse, f;
                if constexpr (CLASSES) {
                    lse = *reinterpret_cast<const f4*>(&at1[buf][16 * i + 4 * g]);
                    f = *reinterpret_cast<const f4*>(&at2[buf][16 * i + 4 * g]);
                } else {
                    lse = f4{own1[u], own1[u], own1[u], own1[u]};
                    f = f4{own2[u], own2[u], own2[u], own2[u]};
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) z[i][u][v] = fast_exp2((z[i][u][v] - lse[v]) * kLog2eF);
                if constexpr (CLASSES) {
                    if (hits) {
                        const u4 at = *reinterpret_cast<const u4*>(&at3[buf][16 * i + 4 * g]);
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            z[i][u][v] -= (int)at[v] == (wave * TILES + u) * 16 + r ? 1.f : 0.f;
                    }
                } else {
                    const int64_t at = t[u] - 64 * c - 16 * i - 4 * g;
                    if (__ballot(at >= 0 && at < 4)) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) z[i][u][v] -= at == v ? 1.f : 0.f;
                    }
                }
                // (0 where f is, whatever z)
#pragma unroll
                for (int v = 0; v < 4; ++v) z[i][u][v] = f[v] == 0.f ? 0.f : z[i][u][v] * f[v];
                if constexpr (CLASSES) sum[u] += (z[i][u][0] + z[i][u][1]) + (z[i][u][2] + z[i][u][3]);
            }
        }
        // times the chunk's rows: their 16 dims from 16 d, rows 32 q + slot_of(g, j)
        v8 dz[2][TILES];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int u = 0; u < TILES; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) dz[q][u][j] = (T)z[2 * q + j / 4][u][j % 4];
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = 32 * q + 4 * g + (r >> 2), at = 2 * (d % 4) + ((r & 3) >> 1);
                const char* from = rows[buf] + d / 4 * kBytes + row * 128 + 16 * (at ^ place_both(row)) +
                                   8 * (r & 1);
                const char* more = rows[buf] + d / 4 * kBytes + (row + 16) * 128 +
                                   16 * (at ^ place_both(row + 16)) + 8 * (r & 1);
                const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)from);
                const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)more);
                const v8 x = __builtin_bit_cast(v8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
#pragma unroll
                for (int u = 0; u < TILES; ++u) acc[u][d] = Half<T>::mfma(x, dz[q][u], acc[u][d]);
            }
    }
    // dims 16 d + 4 g .. of own row r
    const float factor = p.out ? *p.factor : 1.f;
#pragma unroll
    for (int u = 0; u < TILES; ++u) {
        const int64_t row = first + 16 * u + r;
        if (CLASSES && p.sums) {
            float s = sum[u] + __shfl_xor(sum[u], 16, kWave);
            s += __shfl_xor(s, 32, kWave);
            if (g == 0 && row < p.owns) p.sums[blockIdx.y * p.owns + row] = s;
        }
        if (row >= p.owns) continue;
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            const int dim = 16 * d + 4 * g;   // (K is a multiple of 8)
            if (dim >= p.K) continue;
            if (p.out) {
                typedef typename Half<T>::v4 v4;
                struct __attribute__((packed, aligned(2))) Any { v4 v; };
                reinterpret_cast<Any*>(reinterpret_cast<T*>(p.out) + row * p.K + dim)->v =
                    __builtin_convertvector(acc[u][d] * factor, v4);
            } else if (p.slices) {
                *reinterpret_cast<f4*>(p.slices + (blockIdx.y * p.owns + row) * p.K + dim) = acc[u][d];
            }
        }
    }
}

// ---- few classes of few inputs: V <= 64, K <= 256, whole pieces ----
//
// There x's bytes bound the loss, not its products: W stays in LDS in operand order,
// rows stream past it, a row's logits never leave the registers, and the backward pass
// reads x once and writes dx once; dW is summed over a workgroup's rows in registers,
// and the workgroups' sums in order by a second launch.  (200,003 x 128 -> 47 in
// binary16, forward and backward pass by tiles: 33 and 91 us of kernels in 11 launches;
// so 22 and 45 in five.)
constexpr int kFewWaves = 8;
constexpr int64_t kFewClasses = 64, kFewInputs = 256;

struct FewParams {
    const char *x, *w, *bias;
    int64_t ldx;
    const int64_t* target;
    int64_t n, ignore;
    int32_t K, V;
    int32_t reduction;
    float* loss;             // forward
    float* lse;
    double* parts;           // [workgroups][2]
    const float* f;          // backward
    const float* factor;
    char* dx;                // [n][K] or NULL
    float* dw;               // [slices][V][K] or NULL
    float* db;               // [workgroups][V]
};

// W as the first products' operand: fragment f of class tile i, KF fragments a tile.
template <typename T, int KF, int NV>
__device__ __forceinline__ void few_weights(const FewParams& p, typename Half<T>::v8* to)
{
    for (int k = threadIdx.x; k < NV * KF * kWave; k += kFewWaves * kWave) {
        const int l = k % kWave, f = k / kWave % KF, i = k / kWave / KF;
        const int c = 16 * i + (l & 15), at = 32 * f + 8 * (l >> 4);
        typename Half<T>::v8 v = {};
        if (c < p.V && at < p.K)
            v = *reinterpret_cast<const typename Half<T>::v8*>(
                reinterpret_cast<const T*>(p.w) + (int64_t)c * p.K + at);
        to[k] = v;
    }
}
// 16 rows' fragments, dims 32 f + 8 g .. of row r (rows past the last: the last's).
template <typename T, int KF>
__device__ __forceinline__ void few_rows_of(const FewParams& p, int64_t first, int lane,
                                            typename Half<T>::v8 (&x)[KF])
{
    const int g = lane >> 4, r = lane & 15;
    const T* src = reinterpret_cast<const T*>(p.x) + min(first + r, p.n - 1) * p.ldx + 8 * g;
#pragma unroll
    for (int f = 0; f < KF; ++f) {
        x[f] = typename Half<T>::v8{};
        if (32 * f + 8 * g < p.K)
            x[f] = *reinterpret_cast<const typename Half<T>::v8*>(src + 32 * f);
    }
}
// Their logits: classes 16 i + 4 g + v of row r.
template <typename T, int KF, int NV>
__device__ __forceinline__ void few_logits(const typename Half<T>::v8 (&x)[KF],
                                           const typename Half<T>::v8* w, const float* bias,
                                           int lane, f4 (&z)[NV])
{
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        z[i] = *reinterpret_cast<const f4*>(&bias[16 * i + 4 * (lane >> 4)]);
#pragma unroll
        for (int f = 0; f < KF; ++f) z[i] = Half<T>::mfma(w[(i * KF + f) * kWave + lane], x[f], z[i]);
    }
}
template <typename T>
__device__ __forceinline__ void few_bias(const FewParams& p, float* to)
{
    for (int c = threadIdx.x; c < kFewClasses; c += kFewWaves * kWave)
        to[c] = c >= p.V ? -INFINITY : p.bias ? (float)reinterpret_cast<const T*>(p.bias)[c] : 0.f;
}

template <typename T, int KF, int NV>
__global__ void __launch_bounds__(kFewWaves * kWave) few_classes_fwd(const FewParams p)
{
    typedef typename Half<T>::v8 v8;
    __shared__ __align__(16) v8 wl[NV * KF * kWave];
    __shared__ __align__(16) float bl[kFewClasses];
    __shared__ double sums[kFewWaves][2];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int64_t step = (int64_t)gridDim.x * kFewWaves * 16;
    int64_t first = ((int64_t)blockIdx.x * kFewWaves + wave) * 16;
    v8 x[KF], next[KF];
    int64_t t = 0, next_t = 0;
    auto load = [&](int64_t at) __attribute__((always_inline)) {
        few_rows_of<T, KF>(p, at, lane, next);
        next_t = p.target[min(at + r, p.n - 1)];
    };
    load(first);
    few_weights<T, KF, NV>(p, wl);
    few_bias<T>(p, bl);
    __syncthreads();
    double loss = 0.0, counts = 0.0;
    for (; first < p.n; first += step) {
#pragma unroll
        for (int f = 0; f < KF; ++f) x[f] = next[f];
        t = next_t;
        if (first + step < p.n) load(first + step);
        f4 z[NV];
        few_logits<T, KF, NV>(x, wl, bl, lane, z);
        float top = -INFINITY, sum = 0.f, picked = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) top = __builtin_fmaxf(top, z[i][v]);
        top = row_max4(top);
        const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                sum += fast_exp2((z[i][v] - mu) * kLog2eF);
                picked = t == 16 * i + 4 * g + v ? z[i][v] : picked;
            }
        sum += __shfl_xor(sum, 16, kWave);
        sum += __shfl_xor(sum, 32, kWave);
        // (the target's logit, from the lane that has it)
        picked = __shfl(picked, (((int)t >> 2) & 3) * 16 + r, kWave);
        const int64_t row = first + r;
        if (g == 0 && row < p.n) {
            const bool none = t == p.ignore;
            const float l = 0.69314718f * __log2f(sum);
            const float value = none ? 0.f : t < 0 || t >= p.V ? NAN : (top - picked) + l;
            if (p.lse) p.lse[row] = top + l;
            if (p.reduction == kNone) p.loss[row] = value;
            loss += value;
            counts += none ? 0.0 : 1.0;
        }
    }
    loss = wave_sum(loss);
    counts = wave_sum(counts);
    if (lane == 0) {
        sums[wave][0] = loss;
        sums[wave][1] = counts;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        double s = 0.0;
        for (int k = 0; k < kFewWaves; ++k) s += sums[k][threadIdx.x];
        p.parts[2 * (int64_t)blockIdx.x + threadIdx.x] = s;
    }
}

// The operand of a product over rows from a stage of them: 16 columns from 16 t, rows
// 4 g .. and 16 + 4 g .. of the 32 from `at` on.
template <typename T>
__device__ __forceinline__ typename Half<T>::v8 few_columns(const char* at, int stride, int t, int lane)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* lds4;
    const char* from = at + (4 * (lane >> 4) + ((lane & 15) >> 2)) * stride + 32 * t + 8 * (lane & 3);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)from);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(from + 16 * stride));
    return __builtin_bit_cast(typename Half<T>::v8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// 128 rows at a time, 16 a wave: z, dz and dx of a wave's own; then x and dz, through a
// stage of all 128, for the wave's share of dW's dim tiles (with fewer tiles than waves,
// of the rows too: a slice each).  dz is the sum of two 16-bit values (split8): rounded
// once, it added as much to the error of dx and dW as their own rounding.  (200,003 x
// 128 -> 47 trained, kernels: 62 us rounded, 67 so; x 256 -> 47 112 and 120.)
template <typename T, int KF, int NV>
__global__ void __launch_bounds__(kFewWaves * kWave) few_classes_bwd(const FewParams p)
{
    typedef typename Half<T>::v8 v8;
    typedef typename Half<T>::v4 v4;
    constexpr int kTiles = 2 * KF, kFrags = (NV + 1) / 2;   // of dims; of classes, 32 each
    constexpr int kOwn = kTiles >= kFewWaves ? kTiles / kFewWaves : 1;
    constexpr int kSlices = kTiles >= kFewWaves ? 1 : kFewWaves / kTiles;
    // (rows that begin 32 bytes apart modulo 256: eight of them read at once)
    constexpr int kXRow = 64 * KF + 32, kDRow = 32 * NV + (NV > 1 ? 32 : 0);
    // dz's halves lie in LDS side by side, or (256 inputs, 64 classes: 160 KB) in turn
    constexpr int kDBytes = kFewWaves * 16 * kDRow, kInTurn = KF == 8 && NV == 4 ? 2 : 1;
    __shared__ __align__(16) v8 wl[NV * KF * kWave];
    __shared__ __align__(16) v8 wt[kTiles * kFrags * kWave];
    __shared__ __align__(16) float bl[kFewClasses];
    __shared__ __align__(16) char xs[kFewWaves * 16 * kXRow];
    __shared__ __align__(16) char ds[2 / kInTurn * kDBytes];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int64_t step = (int64_t)gridDim.x * kFewWaves * 16;
    int64_t first = (int64_t)blockIdx.x * kFewWaves * 16;   // (of the workgroup)
    v8 x[KF], next[KF];
    int64_t next_t = 0;
    float next_f = 0.f, next_lse = 0.f;
    auto load = [&](int64_t at) __attribute__((always_inline)) {
        at += 16 * wave;
        few_rows_of<T, KF>(p, at, lane, next);
        const int64_t row = min(at + r, p.n - 1);
        next_t = p.target[row];
        next_f = at + r < p.n ? p.f[row] : 0.f;
        next_lse = p.lse[row];
    };
    load(first);
    few_weights<T, KF, NV>(p, wl);
    few_bias<T>(p, bl);
    // W transposed, the classes in the order in which a lane holds a row's dz
    for (int k = threadIdx.x; k < kTiles * kFrags * kWave; k += kFewWaves * kWave) {
        const int l = k % kWave, f = k / kWave % kFrags, dim = 16 * (k / kWave / kFrags) + (l & 15);
        v8 v = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = 32 * f + slot_of(l >> 4, j);
            if (c < p.V && dim < p.K) v[j] = reinterpret_cast<const T*>(p.w)[(int64_t)c * p.K + dim];
        }
        wt[k] = v;
    }
    __syncthreads();
    const float factor = *p.factor;
    f4 dw[kOwn][NV], db[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        db[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < kOwn; ++u) dw[u][i] = f4{0.f, 0.f, 0.f, 0.f};
    }
    char* own_x = xs + wave * 16 * kXRow;
    char* own_d = ds + wave * 16 * kDRow;
    for (; first < p.n; first += step) {
#pragma unroll
        for (int f = 0; f < KF; ++f) x[f] = next[f];
        const int64_t t = next_t;
        const float f = next_f, lse = next_lse;
        if (kInTurn == 1 && first + step < p.n) load(first + step);
        f4 z[NV];
        few_logits<T, KF, NV>(x, wl, bl, lane, z);
        // as the sum of two 16-bit values
        v8 dz[2][kFrags];
        float whole[kFrags][8] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                float d = fast_exp2((z[i][v] - lse) * kLog2eF);
                if (t == 16 * i + 4 * g + v) d -= 1.f;
                d = f == 0.f ? 0.f : d * f;
                if (NV * 16 > p.V && 16 * i + 4 * g + v >= p.V) d = 0.f;   // (f may be NaN)
                db[i][v] += d;
                whole[i / 2][4 * (i & 1) + v] = d;
            }
        }
#pragma unroll
        for (int k = 0; k < kFrags; ++k) split8<T>(whole[k], dz[0][k], dz[1][k]);
        if (p.dw) {
#pragma unroll
            for (int k = 0; k < KF; ++k)   // (rows past the last: with dz of 0, and finite)
                *reinterpret_cast<v8*>(own_x + r * kXRow + 64 * k + 16 * g) =
                    first + 16 * wave + r < p.n ? x[k] : v8{};
        }
        // (registers: behind the logits, where x is done with)
        if (kInTurn > 1 && first + step < p.n) load(first + step);
#pragma unroll
        for (int turn = 0; turn < (p.dw ? kInTurn : 0); ++turn) {
#pragma unroll
            for (int half = 0; half < 2 / kInTurn; ++half)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const v8 of = dz[kInTurn > 1 ? turn : half][i / 2];
                    *reinterpret_cast<v4*>(own_d + half * kDBytes + r * kDRow + 2 * (16 * i + 4 * g)) =
                        (i & 1) ? __builtin_shufflevector(of, of, 4, 5, 6, 7)
                                : __builtin_shufflevector(of, of, 0, 1, 2, 3);
                }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kOwn; ++u) {
                const int tile = kSlices > 1 ? wave % kTiles : wave + u * kFewWaves;
                constexpr int kParts = kFewWaves / 2 / kSlices;   // of 32 rows
#pragma unroll
                for (int q = 0; q < kParts; ++q) {
                    const int rows = 32 * ((kSlices > 1 ? wave / kTiles * kParts : 0) + q);
                    const v8 b = few_columns<T>(xs + rows * kXRow, kXRow, tile, lane);
#pragma unroll
                    for (int half = 0; half < 2 / kInTurn; ++half)
#pragma unroll
                        for (int i = 0; i < NV; ++i)
                            dw[u][i] = Half<T>::mfma(
                                few_columns<T>(ds + half * kDBytes + rows * kDRow, kDRow, i, lane), b,
                                dw[u][i]);
                }
            }
            __syncthreads();
        }
        if (p.dx) {
            // dims 16 t + 4 g .. of row r, whole lines through the wave's part of the stage
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                f4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kFrags; ++k) {
                    const v8 w = wt[(tile * kFrags + k) * kWave + lane];
                    d = Half<T>::mfma(w, dz[0][k], d);
                    d = Half<T>::mfma(w, dz[1][k], d);
                }
                *reinterpret_cast<v4*>(own_x + r * kXRow + 2 * (16 * tile + 4 * g)) =
                    __builtin_convertvector(d * factor, v4);
            }
            wave_lds_order();
            constexpr int kLanes = 4 * KF, kAtOnce = kWave / kLanes;   // per row; rows
#pragma unroll
            for (int v = 0; v < 16 / kAtOnce; ++v) {
                const int rr = v * kAtOnce + lane / kLanes, piece = lane % kLanes;
                const v8 y = *reinterpret_cast<const v8*>(own_x + rr * kXRow + 16 * piece);
                const int64_t row = first + 16 * wave + rr;
                if (row < p.n && 8 * piece < p.K)
                    *reinterpret_cast<v8*>(reinterpret_cast<T*>(p.dx) + row * p.K + 8 * piece) = y;
            }
            wave_lds_order();
        }
    }
    if (p.dw) {
        const int64_t slice = (int64_t)blockIdx.x * kSlices + (kSlices > 1 ? wave / kTiles : 0);
#pragma unroll
        for (int u = 0; u < kOwn; ++u) {
            const int dim = 16 * (kSlices > 1 ? wave % kTiles : wave + u * kFewWaves) + r;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int c = 16 * i + 4 * g + v;
                    if (c < p.V && dim < p.K) p.dw[(slice * p.V + c) * p.K + dim] = dw[u][i][v];
                }
        }
    }
    if (p.db) {
        __syncthreads();
        float* sums = reinterpret_cast<float*>(xs);   // [waves][classes]
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                float s = db[i][v];
#pragma unroll
                for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor(s, off, kWave);
                if (r == 0) sums[wave * kFewClasses + 16 * i + 4 * g + v] = s;
            }
        __syncthreads();
        const int c = threadIdx.x;
        if (c < p.V) {
            float s = 0.f;
            for (int k = 0; k < kFewWaves; ++k) s += sums[k * kFewClasses + c];
            p.db[(int64_t)blockIdx.x * p.V + c] = s;
        }
    }
}

// dW and db from the slices, times the factor: 16 values by 16 parts of the slices.
template <typename T>
__global__ void __launch_bounds__(256)
few_join(const float* __restrict__ dw, int64_t count, int32_t slices, T* __restrict__ out,
         const float* __restrict__ db, int64_t classes, int32_t groups, T* __restrict__ out_db,
         const float* __restrict__ factor)
{
    __shared__ float lds[16][17];
    const int t = threadIdx.x % 16, part = threadIdx.x / 16;
    const int64_t i = (int64_t)blockIdx.x * 16 + t;
    const bool is_db = i >= count;
    const int64_t at = is_db ? i - count : i, stride = is_db ? classes : count;
    const int32_t many = is_db ? groups : slices, per = (many + 15) / 16;
    const int32_t first = min(many, part * per), end = min(many, first + per);
    float s = 0.f;
    if (i < count + classes) s = split_sum((is_db ? db : dw) + at, stride, first, end);
    lds[part][t] = s;
    __syncthreads();
    if (part || i >= count + classes) return;
    for (int k = 1; k < 16; ++k) s += lds[k][t];
    s *= *factor;
    if (is_db) out_db[at] = (T)s;
    else out[at] = (T)s;
}

// Rows of K 16-bit values, as rows of Kp with zeros at their ends, eight a thread; and back.
__global__ void __launch_bounds__(256)
pad_rows(const uint16_t* __restrict__ from, int64_t ld, uint16_t* __restrict__ to, int64_t rows,
         int32_t K, int32_t Kp)
{
    typedef uint16_t v8 __attribute__((ext_vector_type(8)));
    const int32_t pieces = Kp / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces;
         i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / pieces;
        const int32_t c = (int32_t)(i % pieces) * 8;
        const uint16_t* src = from + row * ld + c;
        v8 v = {};
        if (c + 8 <= K) v = reinterpret_cast<const Unaligned<v8>*>(src)->v;
        else
            for (int k = 0; k < K - c; ++k) v[k] = src[k];
        *reinterpret_cast<v8*>(to + row * Kp + c) = v;
    }
}
__global__ void __launch_bounds__(256)
unpad_rows(const uint16_t* __restrict__ from, uint16_t* __restrict__ to, int64_t rows, int32_t K,
           int32_t Kp)
{
    typedef uint16_t v8 __attribute__((ext_vector_type(8)));
    const int32_t pieces = Kp / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces;
         i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / pieces;
        const int32_t c = (int32_t)(i % pieces) * 8;
        const v8 v = *reinterpret_cast<const v8*>(from + row * Kp + c);
        uint16_t* dst = to + row * K + c;
        if (c + 8 <= K) reinterpret_cast<Unaligned<v8>*>(dst)->v = v;
        else
            for (int k = 0; k < K - c; ++k) dst[k] = v[k];
    }
}

__global__ void warm_loss_kernel() {}

hipError_t warm_loss(hipStream_t s)
{
    hipLaunchKernelGGL(warm_loss_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------ launches

struct CeArgs {
    const char *X, *W, *bias;
    int64_t ldx;
    const int64_t* target;
    int64_t ignore;
    int64_t n, K, V;
    int32_t reduction;
    hipStream_t st;
};

// Workgroups of 256 for so many values, below a grid's limit of threads.
static unsigned element_groups(int64_t count)
{
    return (unsigned)std::min<int64_t>(ceil_div(count, 256), 1 << 20);
}

static Tiling one_split(int64_t rows, int64_t outs, int64_t depth, bool odd)
{
    return tiling(rows, outs, depth, depth + 1, odd, false);
}

static bool takes_few(const CeArgs& a)
{
    return a.V <= kFewClasses && a.K <= kFewInputs && a.K % 8 == 0;
}
static int64_t few_groups(int64_t n, bool backward)
{
    return std::min<int64_t>(ceil_div(n, kFewWaves * 16), backward ? 256 : 512);
}
// Slices of dW: those of a workgroup times the workgroups.
static int64_t few_slices(int64_t n, int64_t K)
{
    return few_groups(n, true) * (K <= 64 ? 2 : 1);
}
static FewParams few_params(const CeArgs& a)
{
    FewParams p{};
    p.x = a.X;
    p.w = a.W;
    p.bias = a.bias;
    p.ldx = a.ldx;
    p.target = a.target;
    p.n = a.n;
    p.ignore = a.ignore;
    p.K = (int32_t)a.K;
    p.V = (int32_t)a.V;
    p.reduction = a.reduction;
    return p;
}
template <typename T, bool BACKWARD>
static void launch_few(const FewParams& p, hipStream_t st)
{
    const dim3 grid((unsigned)few_groups(p.n, BACKWARD)), block(kFewWaves * kWave);
    auto go = [&](auto kf, auto nv) {
        constexpr int KF = decltype(kf)::value, NV = decltype(nv)::value;
        if constexpr (BACKWARD) hipLaunchKernelGGL((few_classes_bwd<T, KF, NV>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((few_classes_fwd<T, KF, NV>), grid, block, 0, st, p);
    };
    auto of_k = [&](auto nv) {
        if (p.K <= 64) go(std::integral_constant<int, 2>{}, nv);
        else if (p.K <= 128) go(std::integral_constant<int, 4>{}, nv);
        else go(std::integral_constant<int, 8>{}, nv);
    };
    if (p.V <= 16) of_k(std::integral_constant<int, 1>{});
    else if (p.V <= 32) of_k(std::integral_constant<int, 2>{});
    else of_k(std::integral_constant<int, 4>{});
}

// Chunks of 64 streamed rows in a share, for `groups` workgroups of which `slots` run at
// once: the least rounds of shares, whose starts and ends are some two chunks, and whose
// results `cost` chunks where there are several; `most` shares at most.  (By this and with
// one round's groups at most, us: 52,802 x 64 -> 10,778 672 and 687 trained; 272,567 x 128
// -> 23,790 1,906 and 2,413 forward, 8,849 and 10,017 trained; 70,000 x 64 -> 5,000 422 and
// 482 trained.)
static int64_t share_of(int64_t groups, int64_t chunks, int64_t slots, double cost, int64_t most)
{
    most = std::max<int64_t>(1, std::min(most, chunks));
    int64_t best = chunks;
    double least = INFINITY;
    auto look = [&](int64_t shares) {
        const int64_t per = ceil_div(chunks, std::min(most, std::max<int64_t>(1, shares)));
        shares = ceil_div(chunks, per);
        const double t = (double)ceil_div(groups * shares, slots) * (double)(per + 2) +
                         (shares > 1 ? cost * (double)shares : 0.0);
        if (t < least) {
            least = t;
            best = per;
        }
    };
    for (int64_t k = 1; k <= 8; ++k) look(k);
    for (int64_t k = 1; k <= 4; ++k) look(k * slots / groups);
    return best;
}

static bool streams(int64_t K) { return K <= kFewInputs && K % 8 == 0; }
// (by their LDS; four, two per CU)
static int64_t stream_slots(int64_t K) { return K <= 128 ? 1024 : 512; }

// Workspace of a forward pass: the workgroups' sums, z at the targets, the blocks: one a
// share of the classes, or of as many rows at a time as kBlocksBytes hold.
struct ForwardSpace {
    size_t picked = 0, blocks = 0, bytes = 0;
    int64_t rows = 0, nblocks = 0, per = 0;
};
static ForwardSpace forward_space(int64_t n, int64_t K, int64_t V)
{
    ForwardSpace s;
    if (streams(K)) {
        const int64_t chunks = ceil_div(V, 64);
        s.per = share_of(ceil_div(n, kStreamRows), chunks, stream_slots(K), 0.0, chunks);
        s.nblocks = ceil_div(chunks, s.per);
        s.rows = n;
    } else {
        s.nblocks = ceil_div(V, 32) + 8;   // (at most: the smallest blocks, and a tile's last ones)
        s.rows = std::max<int64_t>(1024, kBlocksBytes / 8 / s.nblocks / 1024 * 1024);
        s.rows = std::min(s.rows, n);
    }
    s.picked = up256(sizeof(double) * 2 * (size_t)ceil_div(n, 4));
    s.blocks = s.picked + up256(sizeof(float) * (size_t)s.rows);
    s.bytes = s.blocks + up256(sizeof(float2) * (size_t)s.rows * s.nblocks);
    return s;
}

template <typename T>
static void launch_stream(const CeArgs& a, const GemmParams& g, int64_t per, int64_t shares)
{
    StreamParams p{};
    p.x = g.P;
    p.w = a.W;
    p.bias = a.bias;
    p.ldx = a.ldx;
    p.rows = g.rows;
    p.V = a.V;
    p.K = (int32_t)a.K;
    p.per = per;
    p.target = g.loss.target;
    p.blocks = g.loss.blocks;
    p.picked = g.loss.picked;
    const dim3 grid((unsigned)ceil_div(p.rows, kStreamRows), (unsigned)shares),
        block(kStreamWaves * kWave);
    if (a.K <= 64) hipLaunchKernelGGL((stream_lse_kernel<T, 1>), grid, block, 0, a.st, p);
    else if (a.K <= 128) hipLaunchKernelGGL((stream_lse_kernel<T, 2>), grid, block, 0, a.st, p);
    else hipLaunchKernelGGL((stream_lse_kernel<T, 4>), grid, block, 0, a.st, p);
}

// Shares of the streamed rows.  A chunk takes some 2.2 us, an output's slice 8 bytes at
// 4 TB/s, written and read.  The slices, float32, are kSliceBytes at most.
constexpr int64_t kSliceBytes = 512 << 20;
constexpr int64_t kGradSlots = 512;   // two per CU
static int64_t grad_rows(int64_t K) { return K <= 128 ? 128 : 64; }   // of a workgroup's own
static int64_t grad_per(int64_t owns, int64_t others, int64_t K)
{
    return share_of(ceil_div(owns, grad_rows(K)), ceil_div(others, 64), kGradSlots,
                    (double)owns * (double)K * (8 / 4e6 / 2.2), kSliceBytes / (owns * K * 4));
}
static int64_t grad_shares(int64_t owns, int64_t others, int64_t K)
{
    return ceil_div(ceil_div(others, 64), grad_per(owns, others, K));
}
template <typename T, bool CLASSES>
static void launch_grad(const GradParams& p, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div(p.owns, grad_rows(p.K)),
                    (unsigned)grad_shares(p.owns, p.others, p.K)),
        block(kStreamWaves * kWave);
    if (p.K <= 64) hipLaunchKernelGGL((stream_grad_kernel<T, 1, 2, CLASSES>), grid, block, 0, st, p);
    else if (p.K <= 128)
        hipLaunchKernelGGL((stream_grad_kernel<T, 2, 2, CLASSES>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((stream_grad_kernel<T, 4, 1, CLASSES>), grid, block, 0, st, p);
}

static int32_t blocks_of(int32_t tile, int64_t outs)
{
    return (int32_t)(ceil_div(outs, tile) * (tile == 256 ? 4 : 2));
}

template <typename T>
static f3s_status loss_forward(const CeArgs& a, float* loss, float* lse, char* ws)
{
    const ForwardSpace s = forward_space(a.n, a.K, a.V);
    CeParams c{};
    c.target = a.target;
    c.n = a.n;
    c.V = a.V;
    c.ignore = a.ignore;
    c.blocks = reinterpret_cast<const float2*>(ws + s.blocks);
    c.picked = reinterpret_cast<const float*>(ws + s.picked);
    c.lse = lse;
    c.loss = loss;
    c.parts = reinterpret_cast<double*>(ws);
    c.reduction = a.reduction;
    if (takes_few(a)) {
        FewParams p = few_params(a);
        p.loss = loss;
        p.lse = lse;
        p.parts = c.parts;
        c.nparts = few_groups(a.n, false);
        launch_few<T, false>(p, a.st);
        if (a.reduction != kNone || lse)
            hipLaunchKernelGGL(loss_total, dim3(1), dim3(1024), 0, a.st, c);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    const bool stream = streams(a.K);
    c.nblocks = stream ? s.nblocks : ceil_div(a.V, 64);   // (or twice as many)
    // Rows per workgroup of a join; the rows of a piece are a multiple of 1,024.
    const int join = c.nblocks <= 16 && a.n >= 4096 ? 256 : a.n <= 2048 ? 4 : 16;
    c.nparts = ceil_div(a.n, join);
    for (int64_t r0 = 0; r0 < a.n; r0 += s.rows) {
        GemmParams p{};
        p.P = a.X + r0 * a.ldx * 2;
        p.ldp = a.ldx;
        p.Q = a.W;
        p.ldq = a.K;
        p.rows = std::min(s.rows, a.n - r0);
        p.outs = a.V;
        p.depth = a.K;
        p.bias = a.bias;
        p.loss.target = a.target + r0;
        p.loss.blocks = reinterpret_cast<float2*>(ws + s.blocks);
        p.loss.picked = reinterpret_cast<float*>(ws + s.picked);
        if (stream) {
            launch_stream<T>(a, p, s.per, c.nblocks);
        } else {
            const bool whole = a.K % 8 == 0;
            const int32_t tile = tile_size(one_split(p.rows, p.outs, p.depth, !whole),
                                           whole ? kWhole : kAny, kEpiLse);
            p.splits = 1;
            if (whole) launch_tiles<T, false, false, kEpiLse, kWhole>(p, tile, a.st);
            else launch_tiles<T, false, false, kEpiLse, kAny>(p, tile, a.st);
            c.nblocks = blocks_of(tile, p.outs);
        }
        F3S_HIP(hipGetLastError());
        c.rows = p.rows;
        c.first_row = r0;
        const dim3 grid((unsigned)ceil_div(p.rows, join));
        if (join == 256) hipLaunchKernelGGL((loss_join<256>), grid, dim3(kLossThreads), 0, a.st, c);
        else if (join == 4) hipLaunchKernelGGL((loss_join<4>), grid, dim3(kLossThreads), 0, a.st, c);
        else hipLaunchKernelGGL((loss_join<16>), grid, dim3(kLossThreads), 0, a.st, c);
    }
    if (a.reduction != kNone || lse)
        hipLaunchKernelGGL(loss_total, dim3(1), dim3(1024), 0, a.st, c);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

constexpr int64_t kLargestGroups = 128;
constexpr int64_t kLossShares = 64;   // of the rows' sums of db

// Workspace of a backward pass: f, the factor, the largest gradients; db's sums; a
// piece's dz; dx's slices; a piece's splits of dW; dW and db of the blocks of rows so far.
struct CeSpace {
    size_t factor = 0, largest = 0, sums = 0, shares = 0, db = 0, dz = 0, dx = 0, dw = 0, bytes = 0;
    size_t few_dw = 0, few_db = 0;   // (few classes)
    size_t all_dw = 0, all_db = 0;   // (several blocks)
    int64_t rows = 0;                // of a block
    int64_t piece = 0, ldz = 0, sum_rows = 0;
    Tiling prob{}, tdx{}, tdw{};
    bool whole_dx = false;   // one piece, one split: dx is written at once
};
// Where dz stays in registers: db's shares, and the slices of dx, then of dW.
struct GradSpace {
    size_t sums = 0, slices = 0, bytes = 0;
};
static GradSpace grad_space(int64_t n, int64_t K, int64_t V, size_t begin)
{
    const int64_t x = grad_shares(n, V, K), w = grad_shares(V, n, K);
    GradSpace s;
    s.sums = begin;
    s.slices = s.sums + up256(sizeof(float) * (size_t)w * V);
    s.bytes = s.slices + up256(sizeof(float) * (size_t)std::max(x > 1 ? x * n * K : 0,
                                                                w > 1 ? w * V * K : 0));
    return s;
}
static CeSpace ce_space(int64_t n, int64_t K, int64_t V)
{
    CeSpace s;
    s.factor = up256(sizeof(float) * (size_t)n);
    s.largest = s.factor + 256;
    s.sums = s.largest + up256(sizeof(float) * kLargestGroups);
    const bool odd = K % 8 != 0;
    if (!odd && V <= kFewClasses && K <= kFewInputs) {
        s.few_dw = s.sums;
        s.few_db = s.few_dw + up256(sizeof(float) * (size_t)few_slices(n, K) * V * K);
        s.bytes = s.few_db + up256(sizeof(float) * (size_t)few_groups(n, true) * V);
        return s;
    }
    if (!odd && K <= kFewInputs) {
        s.bytes = grad_space(n, K, V, s.sums).bytes;
        return s;
    }
    const int64_t blocks = ceil_div(n, kPieceRows);
    s.rows = blocks == 1 ? n : ceil_div(ceil_div(n, blocks), 256) * 256;
    const int64_t fit = kPieceBytes / 2 / s.rows / 256 * 256, pieces = ceil_div(V, fit);
    s.piece = pieces == 1 ? V : ceil_div(ceil_div(V, pieces), 256) * 256;
    s.ldz = ceil_div(s.piece, 8) * 8;
    s.prob = one_split(s.rows, s.ldz, K, odd);
    s.tdx = tiling(s.rows, K, s.piece, kForwardLeast, odd, false);
    s.tdw = tiling(s.piece, K, s.rows, kWeightLeast, odd, true);
    s.whole_dx = s.piece >= V && s.tdx.splits == 1;
    s.sum_rows = 2 * ceil_div(s.rows, 64);   // (at most)
    s.shares = s.sums + up256(sizeof(float) * (size_t)s.sum_rows * s.ldz);
    s.db = s.shares + up256(sizeof(float) * (size_t)kLossShares * s.ldz);
    s.dz = s.db + up256(sizeof(float) * (size_t)s.ldz);
    s.dx = s.dz + up256(2 * (size_t)s.rows * s.ldz);
    s.dw = s.dx + (s.whole_dx ? 0 : up256(sizeof(float) * (size_t)s.tdx.splits * s.rows * K));
    s.all_dw = s.dw + (s.tdw.splits > 1 || blocks > 1
                           ? up256(sizeof(float) * (size_t)s.tdw.splits * s.piece * K)
                           : 0);
    s.all_db = s.all_dw + (blocks > 1 ? up256(sizeof(float) * (size_t)V * K) : 0);
    s.bytes = s.all_db + (blocks > 1 ? up256(sizeof(float) * (size_t)V) : 0);
    return s;
}

// Rows of K inputs that are no whole pieces are copied to ones that are, padded with
// zeros, where the products are long beside that.  (bfloat16, as they are and copied, us:
// 52,802 x 65 -> 10,778 forward 710 and 258, trained 3,051 and 924; x 301 1,059 and 648,
// 5,768 and 2,945; 1,000 x 301 -> 10,000 46 and 42, trained 186 and 158; 3,000 x 301 ->
// 1,000 18.6 and 22.2; 64 x 41 -> 50,021 21.5 and 21.9; 1 x 41 -> 70 15 and 21.)
static bool pads(int64_t n, int64_t K, int64_t V)
{
    return K % 8 != 0 && K < (1 << 22) - 8 && n >= 1000 && n * V >= (1 << 23);
}
struct PadSpace {
    size_t x = 0, w = 0, dx = 0, dw = 0, bytes = 0;
};
static PadSpace pad_space(int64_t n, int64_t K, int64_t V, bool backward)
{
    const int64_t Kp = ceil_div(K, 8) * 8;
    PadSpace s;
    const bool copies = pads(n, K, V);
    s.bytes = backward ? ce_space(n, copies ? Kp : K, V).bytes
                       : forward_space(n, copies ? Kp : K, V).bytes;
    if (!copies) return s;
    const size_t x = up256(2 * (size_t)n * Kp), w = up256(2 * (size_t)V * Kp);
    s.x = s.bytes;
    s.w = s.x + x;
    s.bytes = s.w + w;
    if (backward) {
        s.dx = s.bytes;
        s.dw = s.dx + x;
        s.bytes = s.dw + w;
    }
    return s;
}
static void launch_pad(const char* from, int64_t ld, char* to, int64_t rows, int64_t K, int64_t Kp,
                       hipStream_t st)
{
    hipLaunchKernelGGL(pad_rows, dim3(element_groups(rows * (Kp / 8))), dim3(256), 0, st,
                       reinterpret_cast<const uint16_t*>(from), ld, reinterpret_cast<uint16_t*>(to),
                       rows, (int32_t)K, (int32_t)Kp);
}
static void launch_unpad(const char* from, char* to, int64_t rows, int64_t K, int64_t Kp,
                         hipStream_t st)
{
    hipLaunchKernelGGL(unpad_rows, dim3(element_groups(rows * (Kp / 8))), dim3(256), 0, st,
                       reinterpret_cast<const uint16_t*>(from), reinterpret_cast<uint16_t*>(to), rows,
                       (int32_t)K, (int32_t)Kp);
}
// `a` on padded copies in the workspace.
static CeArgs on_copies(const CeArgs& a, const PadSpace& s, char* ws)
{
    CeArgs b = a;
    b.K = b.ldx = ceil_div(a.K, 8) * 8;
    b.X = ws + s.x;
    b.W = ws + s.w;
    launch_pad(a.X, a.ldx, ws + s.x, a.n, a.K, b.K, a.st);
    launch_pad(a.W, a.K, ws + s.w, a.V, a.K, b.K, a.st);
    return b;
}

// A product of dz and W or x, whose rows are whole pieces beside the padded dz.
template <typename T, bool PT, int EPI>
static f3s_status launch_of_dz(GemmParams p, const Tiling& t, bool pieces, hipStream_t st)
{
    p.splits = t.splits;
    const int32_t tile = tile_size(t, pieces ? kWhole : kAny, EPI);
    F3S_REQUIRE(ceil_div(p.rows, tile) * ceil_div(p.outs, tile) < ((int64_t)1 << 31),
                "cross entropy: too many tiles");
    if (pieces) launch_tiles<T, PT, true, EPI, kWhole>(p, tile, st);
    else launch_tiles<T, PT, true, EPI, kAny>(p, tile, st);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

template <typename T>
static f3s_status loss_backward(const CeArgs& a, const float* lse, const float* dloss, char* dX,
                                char* dW, char* db, char* ws)
{
    const CeSpace s = ce_space(a.n, a.K, a.V);
    constexpr float kUp = Half<T>::kRange ? 16384.f : 1.f;
    float* factor = reinterpret_cast<float*>(ws + s.factor);
    FactorParams f{};
    f.target = a.target;
    f.n = a.n;
    f.V = a.V;
    f.ignore = a.ignore;
    f.dloss = dloss;
    f.count = lse + a.n;
    f.reduction = a.reduction;
    f.lift = kUp;
    f.f = reinterpret_cast<float*>(ws);
    f.factor = factor;
    if (Half<T>::kRange && a.reduction == kNone) {
        f.many = (int32_t)std::min(kLargestGroups, ceil_div(a.n, 4 * kLossThreads));
        f.largest = reinterpret_cast<const float*>(ws + s.largest);
        hipLaunchKernelGGL(loss_largest, dim3((unsigned)f.many), dim3(kLossThreads), 0, a.st, dloss,
                           a.n, reinterpret_cast<float*>(ws + s.largest));
    }
    hipLaunchKernelGGL(loss_factors, dim3((unsigned)ceil_div(a.n, kLossThreads)), dim3(kLossThreads),
                       0, a.st, f);
    F3S_HIP(hipGetLastError());
    if (takes_few(a)) {
        FewParams p = few_params(a);
        p.lse = const_cast<float*>(lse);
        p.f = f.f;
        p.factor = factor;
        p.dx = dX;
        p.dw = dW ? reinterpret_cast<float*>(ws + s.few_dw) : nullptr;
        p.db = db ? reinterpret_cast<float*>(ws + s.few_db) : nullptr;
        launch_few<T, true>(p, a.st);
        const int64_t count = dW ? a.V * a.K : 0, classes = db ? a.V : 0;
        if (count + classes > 0)
            hipLaunchKernelGGL((few_join<T>), dim3((unsigned)ceil_div(count + classes, 16)), dim3(256),
                               0, a.st, p.dw, count, (int32_t)few_slices(a.n, a.K),
                               reinterpret_cast<T*>(dW), p.db, classes,
                               (int32_t)few_groups(a.n, true), reinterpret_cast<T*>(db), factor);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    if (streams(a.K)) {
        const GradSpace w = grad_space(a.n, a.K, a.V, s.sums);
        auto pass = [&](auto classes, char* out, size_t slices, char* sums_out) -> f3s_status {
            constexpr bool kClasses = decltype(classes)::value;
            GradParams p{};
            p.own = kClasses ? a.W : a.X;
            p.other = kClasses ? a.X : a.W;
            p.ld_own = kClasses ? a.K : a.ldx;
            p.ld_other = kClasses ? a.ldx : a.K;
            p.owns = kClasses ? a.V : a.n;
            p.others = kClasses ? a.n : a.V;
            p.K = (int32_t)a.K;
            p.per = grad_per(p.owns, p.others, a.K);
            p.bias = a.bias;
            p.target = a.target;
            p.lse = lse;
            p.f = f.f;
            p.factor = factor;
            const int64_t shares = grad_shares(p.owns, p.others, a.K), count = p.owns * a.K;
            if (out && shares == 1) p.out = out;
            else if (out) p.slices = reinterpret_cast<float*>(ws + slices);
            p.sums = sums_out ? reinterpret_cast<float*>(ws + w.sums) : nullptr;
            launch_grad<T, kClasses>(p, a.st);
            auto join = [&](const float* parts, int64_t values, char* to) {
                hipLaunchKernelGGL((join_scaled<T>), dim3(element_groups(values)), dim3(256), 0,
                                   a.st, parts, values, (int32_t)shares, factor,
                                   reinterpret_cast<T*>(to));
            };
            if (p.slices) join(p.slices, count, out);
            if (p.sums) join(p.sums, p.owns, sums_out);
            F3S_HIP(hipGetLastError());
            return F3S_OK;
        };
        if (dX) F3S_TRY(pass(std::false_type{}, dX, w.slices, nullptr));
        if (dW || db) F3S_TRY(pass(std::true_type{}, dW, w.slices, db));
        return F3S_OK;
    }
    const bool whole = a.K % 8 == 0;   // (the operands' and the results' rows whole pieces)
    const bool blocks = s.rows < a.n;
    // A piece of the classes, v0 .., over the rows r0 ..
    auto piece = [&](int64_t r0, int64_t rows, int64_t v0) -> f3s_status {
        const bool first = r0 == 0, last = r0 + rows == a.n;
        const int64_t outs = std::min(s.piece, a.V - v0), ldz = ceil_div(outs, 8) * 8;
        const char *x = a.X + r0 * a.ldx * 2, *w = a.W + v0 * a.K * 2;
        // (several blocks) slices of dW or db onto those of the blocks before
        auto onto = [&](const float* parts, int64_t count, int32_t slices, size_t sums, int64_t at,
                        char* out) {
            hipLaunchKernelGGL((join_blocks<T>), dim3(element_groups(count)), dim3(256), 0, a.st, parts,
                               count, slices, reinterpret_cast<float*>(ws + sums) + at, first, last,
                               factor, reinterpret_cast<T*>(out) + at);
        };
        GemmParams p{};
        p.P = x;
        p.ldp = a.ldx;
        p.Q = w;
        p.ldq = a.K;
        p.rows = rows;
        p.outs = ldz;
        p.depth = a.K;
        p.bias = a.bias ? a.bias + v0 * 2 : nullptr;
        p.C = ws + s.dz;
        p.sums = db ? reinterpret_cast<float*>(ws + s.sums) : nullptr;
        p.splits = 1;
        p.loss.target = a.target + r0;
        p.loss.first = v0;
        p.loss.lse = lse + r0;
        p.loss.f = f.f + r0;
        p.loss.outs = outs;
        const int32_t tile = tile_size(s.prob, whole ? kWhole : kAny, kEpiProb);
        F3S_REQUIRE(ceil_div(p.rows, tile) * ceil_div(p.outs, tile) < ((int64_t)1 << 31),
                    "cross entropy: too many tiles");
        if (whole) launch_tiles<T, false, false, kEpiProb, kWhole>(p, tile, a.st);
        else launch_tiles<T, false, false, kEpiProb, kAny>(p, tile, a.st);
        F3S_HIP(hipGetLastError());
        if (db) {
            const float* sums = p.sums;
            int64_t many = 2 * ceil_div(rows, tile);
            const unsigned nx = (unsigned)ceil_div(ldz, 64);
            if (many > 512) {   // shares of them first
                float* shares = reinterpret_cast<float*>(ws + s.shares);
                const int64_t ny = std::min<int64_t>(kLossShares, ceil_div(many, 64));
                hipLaunchKernelGGL((column_sums<float>), dim3(nx, (unsigned)ny), dim3(256), 0, a.st,
                                   sums, many, ldz, shares);
                sums = shares;
                many = ny;
            }
            float* all = reinterpret_cast<float*>(ws + s.db);
            hipLaunchKernelGGL((column_sums<float>), dim3(nx, 1), dim3(256), 0, a.st, sums, many, ldz,
                               all);
            if (blocks)
                onto(all, outs, 1, s.all_db, v0, db);
            else
                hipLaunchKernelGGL((cast_scaled<T>), dim3((unsigned)ceil_div(outs, 256)), dim3(256), 0,
                                   a.st, all, outs, factor, reinterpret_cast<T*>(db) + v0);
            F3S_HIP(hipGetLastError());
        }
        if (dX) {
            GemmParams q{};
            q.P = ws + s.dz;
            q.ldp = ldz;
            q.Q = w;
            q.ldq = a.K;
            q.rows = rows;
            q.outs = a.K;
            q.depth = whole ? ldz : outs;
            q.q_end = outs;
            q.add = v0 > 0;
            q.factor = factor;
            q.C = s.whole_dx ? dX + r0 * a.K * 2 : ws + s.dx;
            if (s.whole_dx)
                F3S_TRY((launch_of_dz<T, false, kEpiScaled>(q, s.tdx, whole, a.st)));
            else
                F3S_TRY((launch_of_dz<T, false, kEpiAdd>(q, s.tdx, whole, a.st)));
        }
        if (dW) {
            GemmParams q{};
            q.P = ws + s.dz;
            q.ldp = ldz;
            q.Q = x;
            q.ldq = a.ldx;
            q.rows = outs;
            q.outs = a.K;
            q.depth = q.q_end = rows;
            q.factor = factor;
            char* dst = dW + v0 * a.K * 2;
            if (s.tdw.splits == 1 && !blocks) {
                q.C = dst;
                F3S_TRY((launch_of_dz<T, true, kEpiScaled>(q, s.tdw, whole, a.st)));
            } else {
                q.C = ws + s.dw;
                F3S_TRY((launch_of_dz<T, true, kEpiPart>(q, s.tdw, whole, a.st)));
                const int64_t count = outs * a.K;
                const float* parts = reinterpret_cast<const float*>(ws + s.dw);
                if (blocks)
                    onto(parts, count, s.tdw.splits, s.all_dw, v0 * a.K, dW);
                else
                    hipLaunchKernelGGL((join_scaled<T>), dim3(element_groups(count)), dim3(256), 0,
                                       a.st, parts, count, s.tdw.splits, factor,
                                       reinterpret_cast<T*>(dst));
                F3S_HIP(hipGetLastError());
            }
        }
        return F3S_OK;
    };
    for (int64_t r0 = 0; r0 < a.n; r0 += s.rows) {
        const int64_t rows = std::min(s.rows, a.n - r0);
        for (int64_t v0 = 0; v0 < a.V; v0 += s.piece) F3S_TRY(piece(r0, rows, v0));
        if (dX && !s.whole_dx) {
            const int64_t count = rows * a.K;
            hipLaunchKernelGGL((join_scaled<T>), dim3(element_groups(count)), dim3(256), 0, a.st,
                               reinterpret_cast<const float*>(ws + s.dx), count, s.tdx.splits, factor,
                               reinterpret_cast<T*>(dX) + r0 * a.K);
            F3S_HIP(hipGetLastError());
        }
    }
    return F3S_OK;
}

// Rows of a multiple of eight inputs: 16-byte addresses, offsets in a tile of 31 bits.
static bool pieces_ok(const void* X, int64_t x_stride, const void* W, const void* dX, const void* dW,
                      int64_t K)
{
    const uintptr_t all = (uintptr_t)X | (uintptr_t)W | (uintptr_t)dX | (uintptr_t)dW;
    return K % 8 != 0 || ((all & 15) == 0 && x_stride % 8 == 0 && x_stride < (1 << 22));
}

static f3s_status check_loss(int64_t n, int64_t K, int64_t V, int32_t reduction, int32_t dtype,
                             const char* who)
{
    if (n < 0 || K < 1 || V < 1 || reduction < F3S_LOSS_NONE || reduction > F3S_LOSS_SUM ||
        (dtype != F3S_F16 && dtype != F3S_BF16)) {
        set_error(std::string(who) + ": bad size, reduction or dtype");
        return F3S_EINVAL;
    }
    if (K >= (1 << 22) || V >= ((int64_t)1 << 30) || n >= ((int64_t)1 << 30)) {
        set_error(std::string(who) + ": K below 2^22, classes and n below 2^30");
        return F3S_EUNSUPPORTED;
    }
    return F3S_OK;
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_cross_entropy_workspace(int64_t n, int64_t K, int64_t V, int32_t backward_pass,
                                       int64_t* bytes)
{
    F3S_REQUIRE(bytes, "f3s_cross_entropy_workspace: NULL pointer");
    F3S_TRY(check_loss(n, K, V, F3S_LOSS_NONE, F3S_F16, "f3s_cross_entropy_workspace"));
    *bytes = (int64_t)(n == 0 ? 0 : pad_space(n, K, V, backward_pass != 0).bytes);
    return F3S_OK;
}

f3s_status f3s_cross_entropy_fwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                                 const uint16_t* bias, const int64_t* target, int64_t ignore_index,
                                 float* loss, float* lse, int64_t n, int64_t K, int64_t V,
                                 int32_t reduction, int32_t dtype, void* workspace,
                                 int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_loss(n, K, V, reduction, dtype, "f3s_cross_entropy_fwd"));
    F3S_REQUIRE((n == 0 && reduction == kNone) || loss, "f3s_cross_entropy_fwd: NULL pointer");
    F3S_REQUIRE(n == 0 || (X && W && target && x_stride >= K),
                "f3s_cross_entropy_fwd: NULL pointer, or a row stride below K");
    F3S_REQUIRE(n == 0 || pieces_ok(X, x_stride, W, nullptr, nullptr, K),
                "f3s_cross_entropy_fwd: K is a multiple of 8, X's and W's rows are not at 16-byte "
                "addresses");
    F3S_REQUIRE(n == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 &&
                           workspace_bytes >= (int64_t)pad_space(n, K, V, false).bytes),
                "f3s_cross_entropy_fwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    if (n == 0) {   // (the mean of nothing is NaN, its sum 0)
        CeParams c{};
        c.loss = loss;
        c.lse = lse;
        c.reduction = reduction;
        hipLaunchKernelGGL(loss_total, dim3(1), dim3(1024), 0, as_stream(stream), c);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    const CeArgs a{reinterpret_cast<const char*>(X), reinterpret_cast<const char*>(W),
                   reinterpret_cast<const char*>(bias), x_stride, target, ignore_index, n, K, V,
                   reduction, as_stream(stream)};
    char* ws = static_cast<char*>(workspace);
    const CeArgs b = pads(n, K, V) ? on_copies(a, pad_space(n, K, V, false), ws) : a;
    if (dtype == F3S_F16) return loss_forward<_Float16>(b, loss, lse, ws);
    return loss_forward<__bf16>(b, loss, lse, ws);
}

f3s_status f3s_cross_entropy_bwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                                 const uint16_t* bias, const int64_t* target, int64_t ignore_index,
                                 const float* lse, const float* dloss, uint16_t* dX, uint16_t* dW,
                                 uint16_t* db, int64_t n, int64_t K, int64_t V, int32_t reduction,
                                 int32_t dtype, void* workspace, int64_t workspace_bytes,
                                 void* stream)
{
    F3S_TRY(check_loss(n, K, V, reduction, dtype, "f3s_cross_entropy_bwd"));
    F3S_REQUIRE(n == 0 || (X && W && target && lse && dloss && x_stride >= K),
                "f3s_cross_entropy_bwd: NULL pointer, or a row stride below K");
    F3S_REQUIRE(n == 0 || pieces_ok(X, x_stride, W, dX, dW, K),
                "f3s_cross_entropy_bwd: K is a multiple of 8, the rows of X, W, dX and dW are not "
                "at 16-byte addresses");
    F3S_REQUIRE(n == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 &&
                           workspace_bytes >= (int64_t)pad_space(n, K, V, true).bytes),
                "f3s_cross_entropy_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    if (n == 0) {
        auto zero = [&](uint16_t* out, int64_t count) {
            if (out)
                hipLaunchKernelGGL((loss_zero<_Float16>), dim3(element_groups(count)), dim3(256), 0, st,
                                   reinterpret_cast<_Float16*>(out), count);
        };
        zero(dW, V * K);
        zero(db, V);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    if (!dX && !dW && !db) return F3S_OK;
    const CeArgs a{reinterpret_cast<const char*>(X), reinterpret_cast<const char*>(W),
                   reinterpret_cast<const char*>(bias), x_stride, target, ignore_index, n, K, V,
                   reduction, st};
    char* ws = static_cast<char*>(workspace);
    char *dx = reinterpret_cast<char*>(dX), *dw = reinterpret_cast<char*>(dW);
    CeArgs b = a;
    const PadSpace pad = pad_space(n, K, V, true);
    if (pads(n, K, V)) {
        b = on_copies(a, pad, ws);
        if (dx) dx = ws + pad.dx;
        if (dw) dw = ws + pad.dw;
    }
    if (dtype == F3S_F16)
        F3S_TRY(loss_backward<_Float16>(b, lse, dloss, dx, dw, reinterpret_cast<char*>(db), ws));
    else
        F3S_TRY(loss_backward<__bf16>(b, lse, dloss, dx, dw, reinterpret_cast<char*>(db), ws));
    if (pads(n, K, V)) {
        if (dX) launch_unpad(dx, reinterpret_cast<char*>(dX), n, K, b.K, st);
        if (dW) launch_unpad(dw, reinterpret_cast<char*>(dW), V, K, b.K, st);
        F3S_HIP(hipGetLastError());
    }
    return F3S_OK;
}

}  // extern "C"
