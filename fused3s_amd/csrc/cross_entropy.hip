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
//            rows of dW.  A piece's dz is kPieceBytes at most.  So memory goes with n, K and that, not with n V, for one product
//            of four more than keeping z would take.
// dz is rounded to the type, the operand that dx and dW take: these two carry that
// rounding beside their own; db is summed before it.  What dz is multiplied with
// throughout (1 / count, a loss scale) comes last, in float32, so that small gradients
// do not vanish: dz itself is of size 1 at most, in binary16 times 2^14, as a class
// of probability 1e-9 still has its 11 bits then.
// What bounds it is the matrix cores, with many classes; with few, x.
#include <cmath>

#include "gemm_tiles.hpp"

namespace f3s {

// (16,384 x 512 -> 100,003, a training step, milliseconds with pieces of 128, 256, 512 and
// 1,024 MB: 8.9, 8.9, 8.5, 9.1: fewer launches and additions of dx against what the
// Infinity Cache holds.)
constexpr int64_t kPieceBytes = 512 << 20;    // of dz
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
// order.  (64 rows of 1,564 blocks, 16 rows a workgroup: 16 us, four: 6; 200,003 rows of
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
        // (kept where its inverse is one too)
        const int e = m > 0.f ? __builtin_amdgcn_frexp_expf(m) : 0;
        unit = __builtin_amdgcn_ldexpf(1.f, e < -120 ? -120 : e > 120 ? 120 : e);
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
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) out[i] = (T)(split_sum(parts + i, count, 0, slices) * *factor);
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
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) out[i] = (T)0.f;
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

static Tiling one_split(int64_t rows, int64_t outs, int64_t depth, bool odd)
{
    return tiling(rows, outs, depth, depth + 1, odd, false);
}

// Workspace of a forward pass: the workgroups' sums, z at the targets, the blocks of as
// many rows at a time as kBlocksBytes hold.
struct ForwardSpace {
    size_t picked = 0, blocks = 0, bytes = 0;
    int64_t rows = 0, nblocks = 0;
};
static ForwardSpace forward_space(int64_t n, int64_t V)
{
    ForwardSpace s;
    s.nblocks = ceil_div(V, 32) + 8;   // (at most: the smallest blocks, and a tile's last ones)
    s.rows = std::max<int64_t>(1024, kBlocksBytes / 8 / s.nblocks / 1024 * 1024);
    s.rows = std::min(s.rows, n);
    s.picked = up256(sizeof(double) * 2 * (size_t)ceil_div(n, 4));
    s.blocks = s.picked + up256(sizeof(float) * (size_t)s.rows);
    s.bytes = s.blocks + up256(sizeof(float2) * (size_t)s.rows * s.nblocks);
    return s;
}

static int32_t blocks_of(int32_t tile, int64_t outs)
{
    return (int32_t)(ceil_div(outs, tile) * (tile == 256 ? 4 : 2));
}

template <typename T>
static f3s_status loss_forward(const CeArgs& a, float* loss, float* lse, char* ws)
{
    const ForwardSpace s = forward_space(a.n, a.V);
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
    // (rows per workgroup of a join; the rows of a piece are a multiple of 1,024)
    const int64_t most = ceil_div(a.V, 64);
    const int join = most <= 16 && a.n >= 4096 ? 256 : a.n <= 2048 ? 4 : 16;
    c.nparts = ceil_div(a.n, join);
    c.reduction = a.reduction;
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
        const Tiling t = one_split(p.rows, p.outs, p.depth, a.K % 8 != 0);
        GemmParams q = p;   // (C is not written, and nothing of bias is read in pieces)
        q.bias = nullptr;
        q.outs = ceil_div(a.V, 8) * 8;
        const Way way = way_of(q) == kAny ? kAny : kWhole;
        const int32_t tile = tile_size(t, way, kEpiLse);
        F3S_REQUIRE(ceil_div(p.rows, tile) * ceil_div(p.outs, tile) < ((int64_t)1 << 31),
                    "cross entropy: too many tiles");
        p.splits = 1;
        if (way == kWhole) launch_tiles<T, false, false, kEpiLse, kWhole>(p, tile, a.st);
        else launch_tiles<T, false, false, kEpiLse, kAny>(p, tile, a.st);
        F3S_HIP(hipGetLastError());
        c.nblocks = blocks_of(tile, p.outs);
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
// piece's dz; dx's slices; a piece's splits of dW.
struct CeSpace {
    size_t factor = 0, largest = 0, sums = 0, shares = 0, db = 0, dz = 0, dx = 0, dw = 0, bytes = 0;
    int64_t piece = 0, ldz = 0, sum_rows = 0;
    Tiling prob{}, tdx{}, tdw{};
    bool whole_dx = false;   // one piece, one split: dx is written at once
};
static CeSpace ce_space(int64_t n, int64_t K, int64_t V)
{
    CeSpace s;
    const bool odd = K % 8 != 0;
    const int64_t fit = std::max<int64_t>(1024, kPieceBytes / 2 / n / 256 * 256);
    const int64_t pieces = ceil_div(V, fit);
    s.piece = pieces == 1 ? V : ceil_div(ceil_div(V, pieces), 256) * 256;
    s.ldz = ceil_div(s.piece, 8) * 8;
    s.prob = one_split(n, s.ldz, K, odd);
    s.tdx = tiling(n, K, s.piece, kForwardLeast, odd, false);
    s.tdw = tiling(s.piece, K, n, kWeightLeast, odd, true);
    s.whole_dx = s.piece >= V && s.tdx.splits == 1;
    s.sum_rows = 2 * ceil_div(n, 64);   // (at most)
    s.factor = up256(sizeof(float) * (size_t)n);
    s.largest = s.factor + 256;
    s.sums = s.largest + up256(sizeof(float) * kLargestGroups);
    s.shares = s.sums + up256(sizeof(float) * (size_t)s.sum_rows * s.ldz);
    s.db = s.shares + up256(sizeof(float) * (size_t)kLossShares * s.ldz);
    s.dz = s.db + up256(sizeof(float) * (size_t)s.ldz);
    s.dx = s.dz + up256(2 * (size_t)n * s.ldz);
    s.dw = s.dx + (s.whole_dx ? 0 : up256(sizeof(float) * (size_t)s.tdx.splits * n * K));
    s.bytes = s.dw +
              (s.tdw.splits > 1 ? up256(sizeof(float) * (size_t)s.tdw.splits * s.piece * K) : 0);
    return s;
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
    auto aligned = [](const void* x) { return ((uintptr_t)x & 15) == 0; };
    const bool w_pieces = a.K % 8 == 0 && a.K < (1 << 22) && aligned(a.W);
    const bool x_pieces = a.K % 8 == 0 && a.ldx % 8 == 0 && a.ldx < (1 << 22) && aligned(a.X);
    for (int64_t v0 = 0; v0 < a.V; v0 += s.piece) {
        const int64_t outs = std::min(s.piece, a.V - v0), ldz = ceil_div(outs, 8) * 8;
        const char* w = a.W + v0 * a.K * 2;
        GemmParams p{};
        p.P = a.X;
        p.ldp = a.ldx;
        p.Q = w;
        p.ldq = a.K;
        p.rows = a.n;
        p.outs = ldz;
        p.depth = a.K;
        p.bias = a.bias ? a.bias + v0 * 2 : nullptr;
        p.C = ws + s.dz;
        p.sums = db ? reinterpret_cast<float*>(ws + s.sums) : nullptr;
        p.splits = 1;
        p.loss.target = a.target;
        p.loss.first = v0;
        p.loss.lse = lse;
        p.loss.f = f.f;
        p.loss.outs = outs;
        const bool pieces = w_pieces && x_pieces;
        const int32_t tile = tile_size(s.prob, pieces ? kWhole : kAny, kEpiProb);
        F3S_REQUIRE(ceil_div(p.rows, tile) * ceil_div(p.outs, tile) < ((int64_t)1 << 31),
                    "cross entropy: too many tiles");
        if (pieces) launch_tiles<T, false, false, kEpiProb, kWhole>(p, tile, a.st);
        else launch_tiles<T, false, false, kEpiProb, kAny>(p, tile, a.st);
        F3S_HIP(hipGetLastError());
        if (db) {
            const float* sums = p.sums;
            int64_t rows = 2 * ceil_div(a.n, tile);
            const unsigned nx = (unsigned)ceil_div(ldz, 64);
            if (rows > 512) {   // shares of them first
                float* shares = reinterpret_cast<float*>(ws + s.shares);
                const int64_t ny = std::min<int64_t>(kLossShares, ceil_div(rows, 64));
                hipLaunchKernelGGL((column_sums<float>), dim3(nx, (unsigned)ny), dim3(256), 0, a.st,
                                   sums, rows, ldz, shares);
                sums = shares;
                rows = ny;
            }
            float* whole = reinterpret_cast<float*>(ws + s.db);
            hipLaunchKernelGGL((column_sums<float>), dim3(nx, 1), dim3(256), 0, a.st, sums, rows, ldz,
                               whole);
            hipLaunchKernelGGL((cast_scaled<T>), dim3((unsigned)ceil_div(outs, 256)), dim3(256), 0,
                               a.st, whole, outs, factor, reinterpret_cast<T*>(db) + v0);
            F3S_HIP(hipGetLastError());
        }
        if (dX) {
            GemmParams q{};
            q.P = ws + s.dz;
            q.ldp = ldz;
            q.Q = w;
            q.ldq = a.K;
            q.rows = a.n;
            q.outs = a.K;
            q.depth = w_pieces ? ldz : outs;
            q.q_end = outs;
            q.add = v0 > 0;
            q.factor = factor;
            q.C = s.whole_dx ? dX : ws + s.dx;
            if (s.whole_dx)
                F3S_TRY((launch_of_dz<T, false, kEpiScaled>(q, s.tdx, w_pieces && aligned(dX), a.st)));
            else
                F3S_TRY((launch_of_dz<T, false, kEpiAdd>(q, s.tdx, w_pieces, a.st)));
        }
        if (dW) {
            GemmParams q{};
            q.P = ws + s.dz;
            q.ldp = ldz;
            q.Q = a.X;
            q.ldq = a.ldx;
            q.rows = outs;
            q.outs = a.K;
            q.depth = q.q_end = a.n;
            q.factor = factor;
            char* dst = dW + v0 * a.K * 2;
            if (s.tdw.splits == 1) {
                q.C = dst;
                F3S_TRY((launch_of_dz<T, true, kEpiScaled>(q, s.tdw, x_pieces && aligned(dst), a.st)));
            } else {
                q.C = ws + s.dw;
                F3S_TRY((launch_of_dz<T, true, kEpiPart>(q, s.tdw, x_pieces, a.st)));
                const int64_t count = outs * a.K;
                hipLaunchKernelGGL((join_scaled<T>), dim3((unsigned)ceil_div(count, 256)), dim3(256),
                                   0, a.st, reinterpret_cast<const float*>(ws + s.dw), count,
                                   s.tdw.splits, factor, reinterpret_cast<T*>(dst));
                F3S_HIP(hipGetLastError());
            }
        }
    }
    if (dX && !s.whole_dx) {
        const int64_t count = a.n * a.K;
        hipLaunchKernelGGL((join_scaled<T>), dim3((unsigned)ceil_div(count, 256)), dim3(256), 0, a.st,
                           reinterpret_cast<const float*>(ws + s.dx), count, s.tdx.splits, factor,
                           reinterpret_cast<T*>(dX));
        F3S_HIP(hipGetLastError());
    }
    return F3S_OK;
}

static f3s_status check_loss(int64_t n, int64_t K, int64_t V, int32_t reduction, int32_t dtype,
                             const char* who)
{
    if (n < 0 || K < 1 || V < 1 || reduction < F3S_LOSS_NONE || reduction > F3S_LOSS_SUM ||
        (dtype != F3S_F16 && dtype != F3S_BF16)) {
        set_error(std::string(who) + ": bad size, reduction or dtype");
        return F3S_EINVAL;
    }
    if (K >= (1 << 22) || V >= ((int64_t)1 << 30) || n >= ((int64_t)1 << 31)) {
        set_error(std::string(who) + ": K below 2^22, classes below 2^30, n below 2^31");
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
    *bytes = (int64_t)(n == 0 ? 0 : backward_pass ? ce_space(n, K, V).bytes : forward_space(n, V).bytes);
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
    F3S_REQUIRE(n == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 &&
                           workspace_bytes >= (int64_t)forward_space(n, V).bytes),
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
    if (dtype == F3S_F16) return loss_forward<_Float16>(a, loss, lse, static_cast<char*>(workspace));
    return loss_forward<__bf16>(a, loss, lse, static_cast<char*>(workspace));
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
    F3S_REQUIRE(n == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 &&
                           workspace_bytes >= (int64_t)ce_space(n, K, V).bytes),
                "f3s_cross_entropy_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    if (n == 0) {
        auto zero = [&](uint16_t* out, int64_t count) {
            if (out)
                hipLaunchKernelGGL((loss_zero<_Float16>), dim3((unsigned)ceil_div(count, 256)),
                                   dim3(256), 0, st, reinterpret_cast<_Float16*>(out), count);
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
    if (dtype == F3S_F16)
        return loss_backward<_Float16>(a, lse, dloss, reinterpret_cast<char*>(dX),
                                       reinterpret_cast<char*>(dW), reinterpret_cast<char*>(db), ws);
    return loss_backward<__bf16>(a, lse, dloss, reinterpret_cast<char*>(dX),
                                 reinterpret_cast<char*>(dW), reinterpret_cast<char*>(db), ws);
}

}  // extern "C"
