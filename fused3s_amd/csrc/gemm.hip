// gemm.hip -- y = act(x W^T + b) + r and its gradient, any sizes, binary16 and
// bfloat16 with float32 sums.
//
// One tiled product serves all three directions: C[row][out] = sum_c P(row, c)
// Q(out, c), where an operand lies row by row ([row][c]) or contraction by
// contraction ([c][row]):
//   forward  P = x [n][K],      Q = W [M][K]
//   dz       the same again, dz = dy act'(z) in its epilogue: z is not kept from
//            the forward pass (n M values of memory and their traffic; in 16 bits
//            its rounding would double dz's).  dz is rounded to the type, the
//            operand that the two products after it take: dx and dW carry that
//            rounding beside their own, 1.41 x the error of one (32,768 x 1,024 ->
//            4,096, gelu, bfloat16, against 64 bits in the 2-norm: 2.34e-3, where
//            rounding the result alone is 1.66e-3).  Two 16-bit values for each
//            would take twice the matrix instructions of both (six products' for a
//            step's four).  db is summed before the rounding.  Without an activation
//            dz is dy, and every result is rounded once.
//   dx       P = dz [n][M],     Q = W, transposed
//   dW       P, Q = dz, x, both transposed, n cut into splits whose float32
//            sums are added in order; db with it
// A workgroup owns a block of C and goes through the contraction in steps: both
// operands' tiles go from memory straight into LDS (16 bytes a lane, no registers),
// ahead of the products, in an order in which neither plain nor transposing LDS
// reads meet bank conflicts.  Q is the MFMA's A operand, so a lane holds four
// consecutive outputs of a row; the epilogue passes them through LDS, 16 rows at a
// time, so that whole lines are read (residual, dy) and written.  Two kernels of
// their own: a few rows, and many rows of few inputs.
#include "gemm_tiles.hpp"

namespace f3s {

// Few rows (one token, a small batch): a workgroup takes 16 outputs, its waves a
// share of the contraction each, W's rows loaded once, straight into operands.
// Bound by the one latency of those loads and the launch, not by their bytes.
template <typename T, int NT, bool FAST>
__global__ void __launch_bounds__(512)
few_rows_kernel(const GemmParams p)
{
    typedef typename Half<T>::v8 v8;
    constexpr int kWaves = 8;
    __shared__ __align__(16) f4 parts[kWaves][NT][kWave];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int64_t out0 = (int64_t)blockIdx.x * 16;
    const T* W = reinterpret_cast<const T*>(p.Q) + min(out0 + r, p.outs - 1) * p.ldq;
    const T* X = reinterpret_cast<const T*>(p.P);
    const int64_t blocks = (p.depth + 31) / 32, per = (blocks + kWaves - 1) / kWaves;
    const int64_t fb = wave * per, fe = min(blocks, fb + per);
    auto load = [&](const T* row, int64_t k) __attribute__((always_inline)) -> v8 {
        v8 v = {};
        if constexpr (FAST) {
            if (k < p.depth) v = *reinterpret_cast<const v8*>(row + k);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < p.depth) v[e] = row[k + e];
        }
        return v;
    };
    f4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    for (int64_t f = fb; f < fe; ++f) {
        const int64_t k = 32 * f + 8 * g;
        const v8 a = load(W, k);
#pragma unroll
        for (int t = 0; t < NT; ++t)
            acc[t] = Half<T>::mfma(a, load(X + min((int64_t)(16 * t + r), p.rows - 1) * p.ldp, k),
                                   acc[t]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) parts[wave][t][lane] = acc[t];
    __syncthreads();
    // a wave finishes row tile t: four outputs of a row per lane
    for (int t = wave; t < NT; t += kWaves) {
        f4 z = parts[0][t][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) z += parts[w][t][lane];
        const int64_t row = 16 * t + r;
        if (row >= p.rows) continue;
        float y[4] = {z[0], z[1], z[2], z[3]};
        const int64_t out = out0 + 4 * g;
        const int many = (int)min((int64_t)4, p.outs - out);
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (p.bias && v < many) y[v] += (float)reinterpret_cast<const T*>(p.bias)[out + v];
        act_values(p.act, y);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            if (v >= many) break;
            if (p.R) y[v] += (float)reinterpret_cast<const T*>(p.R)[row * p.ldr + out + v];
            reinterpret_cast<T*>(p.C)[row * p.outs + out + v] = (T)y[v];
        }
    }
}

// Sums over a row's 16 lanes of eight values each: lane r is left with those of
// values 4 (r & 1) + 2 (r >> 1 & 1) + {0, 1}.
template <int CTRL>
__device__ __forceinline__ float from_lane(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf,
                                                              0xf, true));
}
__device__ __forceinline__ f2 row_sums(const float (&v)[8], int r)
{
    constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kRor4 = 0x124, kRor8 = 0x128;
    float a[4], c[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float keep = r & 1 ? v[k + 4] : v[k], give = r & 1 ? v[k] : v[k + 4];
        a[k] = keep + from_lane<kXor1>(give);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float keep = r & 2 ? a[k + 2] : a[k], give = r & 2 ? a[k] : a[k + 2];
        c[k] = keep + from_lane<kXor2>(give);
        c[k] += from_lane<kRor4>(c[k]);
        c[k] += from_lane<kRor8>(c[k]);
    }
    return f2{c[0], c[1]};
}

// Many rows of few inputs (K <= 256): W (or as many of its columns as 96 KB hold)
// is laid out once per workgroup in LDS, in the order the MFMA operands are read,
// and 16 waves stream blocks of 16 rows past it, their operands loaded straight
// into registers, one block ahead.  W's rows are dealt to the tiles so that a lane
// holds eight consecutive outputs of one row (two 16 x 16 tiles side by side); two
// such pieces go through a small stage so that whole 128-byte lines are stored.
// MODE: act(z + bias), + R, or dy act'(z + bias) and the sums of its columns (a
// wave's own in LDS, joined in order at the end).
// Bound by the rows in and out, and by the activation where it has one (gelu: 20
// operations' time a value).
// (f3s_linear_f16's linear_kernel (linear.hip) streams rows past W in the same order, in
// binary16, without strides or an epilogue; from 48 K rows on both give the same bits.
// It stays for the forward-only layer: 50,000 x 64 -> 192 7.2 us against 8.0 here, where
// the activation is looked at for every piece; 50,000 x 128 -> 384 14.7 and 15.1,
// 500,000 x 128 -> 512 133 and 134; and below 48 K rows its callers keep the bits they
// have, which tiles do not give.)
enum RowsMode : int { kRowsAct = 0, kRowsResidual = 1, kRowsSlope = 2 };
constexpr int kRowWaves = 16, kRowPieces = 6144;
// outputs per workgroup at most
constexpr int rows_cols(int kf, int mode)
{
    const int most = kRowPieces / (4 * kf);
    return mode == kRowsSlope && most > 384 ? 384 : most;   // (the sums: 64 bytes of LDS each)
}
template <typename T, int KF, int MODE>
__global__ void __launch_bounds__(kRowWaves * kWave) __attribute__((amdgpu_waves_per_eu(4)))
rows_kernel(const GemmParams p)
{
    constexpr bool RES = MODE != kRowsAct, SLOPE = MODE == kRowsSlope;
    constexpr int kCols = rows_cols(KF, MODE);
    typedef typename Half<T>::v8 v8;
    __shared__ __align__(16) v8 wl[kRowPieces];
    __shared__ __align__(16) T bl[kCols];
    __shared__ __align__(16) T stage[kRowWaves][16 * kStageRow];
    __shared__ __align__(16) float sums[SLOPE ? kRowWaves : 1][SLOPE ? kCols : 1];
    const int tid = threadIdx.x, lane = tid % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int g = lane >> 4, r = lane & 15;
    const int32_t K = (int32_t)p.depth, M = (int32_t)p.outs;
    const int32_t cols = (int32_t)p.split;   // outputs per workgroup (blockIdx.y)
    const int32_t m0 = blockIdx.y * cols, mc = min(cols, M - m0);   // multiples of 32
    const T* W = reinterpret_cast<const T*>(p.Q);
    const T* X = reinterpret_cast<const T*>(p.P);
    const T* R = reinterpret_cast<const T*>(p.R);
    const T* bias = reinterpret_cast<const T*>(p.bias);
    T* Y = reinterpret_cast<T*>(p.C);
    const v8 zero = {};

    // piece (((pair * 2 + t) * KF + f) * 64 + l) is what lane l supplies for fragment
    // f of tile t of that pair of tiles
    for (int i = tid; i < mc * KF * 4; i += kRowWaves * kWave) {
        const int l = i & 63, f = (i >> 6) % KF, tile = (i >> 6) / KF;
        const int row = l & 15;
        const int col = (tile >> 1) * 32 + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3);
        const int k = 32 * f + 8 * (l >> 4);
        v8 w = zero;
        if (k < K && !p.q_steps) {
            w = *reinterpret_cast<const v8*>(W + (int64_t)(m0 + col) * p.ldq + k);
        } else if (k < K) {   // (dx; once per workgroup)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = W[(k + e) * p.ldq + m0 + col];
        }
        wl[i] = w;
    }
    for (int i = tid; i < mc; i += kRowWaves * kWave) bl[i] = bias ? bias[m0 + i] : (T)0.f;
    if constexpr (SLOPE)
        for (int i = tid; i < kRowWaves * kCols; i += kRowWaves * kWave) sums[0][i] = 0.f;
    __syncthreads();

    const int64_t blocks = (p.rows + 15) >> 4, step = (int64_t)gridDim.x * kRowWaves;
    int64_t b = (int64_t)blockIdx.x * kRowWaves + wave;
    if (!SLOPE && b >= blocks) return;
    auto load = [&](int64_t blk, v8 (&x)[KF]) __attribute__((always_inline)) {
        const int64_t row = min(blk * 16 + r, p.rows - 1);   // (past the end: not stored)
        const T* src = X + row * p.ldp + 8 * g;
#pragma unroll
        for (int f = 0; f < KF; ++f)
            x[f] = 32 * f + 8 * g < K ? *reinterpret_cast<const v8*>(src + 32 * f) : zero;
    };
    v8 x[KF], nx[KF], res[2];
    // outputs c + 8 g .. + 7 of row r of the block
    auto product = [&](int32_t c, v8 rest) __attribute__((always_inline)) -> v8 {
        typedef float f8 __attribute__((ext_vector_type(8)));
        const v8* w = wl + (c >> 5) * (2 * KF * 64) + lane;
        const f8 bf = __builtin_convertvector(*reinterpret_cast<const v8*>(&bl[c + 8 * g]), f8);
        f4 a0 = {bf[0], bf[1], bf[2], bf[3]}, a1 = {bf[4], bf[5], bf[6], bf[7]};
#pragma unroll
        for (int f = 0; f < KF; ++f) {
            a0 = Half<T>::mfma(w[f * 64], x[f], a0);
            a1 = Half<T>::mfma(w[(KF + f) * 64], x[f], a1);
        }
        float y[8] = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
        if constexpr (SLOPE) {
            float dy[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) dy[k] = (float)rest[k];
            act_gradients(p.act, y, dy);
            if (p.sums) {
                float own[8];   // (a row past the end repeats the last one)
#pragma unroll
                for (int k = 0; k < 8; ++k) own[k] = b * 16 + r < p.rows ? y[k] : 0.f;
                const f2 s = row_sums(own, r);
                if (r < 4) {
                    f2* to = reinterpret_cast<f2*>(&sums[wave][c + 8 * g + 4 * (r & 1) + (r & 2)]);
                    *to = f2{(*to)[0] + s[0], (*to)[1] + s[1]};
                }
            }
        } else {
            act_values(p.act, y);
        }
        if constexpr (MODE == kRowsResidual) {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] += (float)rest[k];
        }
        return __builtin_convertvector((f8{y[0], y[1], y[2], y[3], y[4], y[5], y[6], y[7]}), v8);
    };
    auto residual = [&](int64_t blk, int32_t c) __attribute__((always_inline)) -> v8 {
        const int64_t row = min(blk * 16 + r, p.rows - 1);
        return *reinterpret_cast<const v8*>(R + row * p.ldr + m0 + c + 8 * g);
    };
    T* out = stage[wave];
    load(b, x);
    if constexpr (RES) {
        res[0] = residual(b, 0);
        if (mc >= 64) res[1] = residual(b, 32);
    }
    for (; b < blocks; b += step) {
        const bool more = b + step < blocks;
        if (more) load(b + step, nx);
        int32_t c = 0;
        for (; c + 64 <= mc; c += 64) {
            const v8 now0 = res[0], now1 = res[1];
            if constexpr (RES) {   // the next 64 columns', or the next block's first
                const int32_t cn = c + 64 < mc ? c + 64 : 0;
                if (cn || more) {
                    const int64_t bn = cn ? b : b + step;
                    res[0] = residual(bn, cn);
                    if (cn + 64 <= mc) res[1] = residual(bn, cn + 32);
                }
            }
            *reinterpret_cast<v8*>(&out[r * kStageRow + 8 * g]) = product(c, now0);
            *reinterpret_cast<v8*>(&out[r * kStageRow + 32 + 8 * g]) = product(c + 32, now1);
            wave_lds_order();
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int rr = 8 * v + (lane >> 3);
                const v8 y = *reinterpret_cast<const v8*>(&out[rr * kStageRow + 8 * (lane & 7)]);
                const int64_t row = b * 16 + rr;
                if (row < p.rows) *reinterpret_cast<v8*>(Y + row * M + m0 + c + 8 * (lane & 7)) = y;
            }
            wave_lds_order();
        }
        if (c < mc) {   // 32 columns are left
            const v8 now0 = res[0];
            if (RES && more) {
                res[0] = residual(b + step, 0);
                if (mc >= 64) res[1] = residual(b + step, 32);
            }
            const v8 y = product(c, now0);
            if (b * 16 + r < p.rows)
                *reinterpret_cast<v8*>(Y + (b * 16 + r) * M + m0 + c + 8 * g) = y;
        }
#pragma unroll
        for (int f = 0; f < KF; ++f) x[f] = nx[f];
    }
    if constexpr (SLOPE) {
        __syncthreads();
        if (p.sums && tid < mc) {
            float s = 0.f;
            for (int w = 0; w < kRowWaves; ++w) s += sums[w][tid];
            p.sums[(int64_t)blockIdx.x * M + m0 + tid] = s;
        }
    }
}

// The same for the slope pass: dz, and the sums of the columns of blockIdx.y's share
// of the rows; 64 columns per workgroup.
template <typename T>
__global__ void __launch_bounds__(256)
join_slope(const GemmParams p, const float* __restrict__ parts)
{
    __shared__ float lds[4][64];
    const int64_t col = (int64_t)blockIdx.x * 64 + threadIdx.x % 64, count = p.rows * p.outs;
    const int part = threadIdx.x / 64;
    const int64_t per = (p.rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = blockIdx.y * per, r1 = min(p.rows, r0 + per);
    float sum = 0.f;
    if (col < p.outs) {
        const float bias = p.bias ? (float)reinterpret_cast<const T*>(p.bias)[col] : 0.f;
        for (int64_t row = r0 + part; row < r1; row += 4) {
            float z[1] = {0.f};
            for (int32_t k = 0; k < p.splits; ++k) z[0] += parts[k * count + row * p.outs + col];
            z[0] += bias;
            const float dy[1] = {(float)reinterpret_cast<const T*>(p.R)[row * p.ldr + col]};
            act_gradients(p.act, z, dy);
            sum += z[0];
            reinterpret_cast<T*>(p.C)[row * p.outs + col] = (T)z[0];
        }
    }
    lds[part][threadIdx.x % 64] = sum;
    __syncthreads();
    if (p.sums && part == 0 && col < p.outs) {
        const int t = threadIdx.x;
        p.sums[blockIdx.y * p.outs + col] = (lds[0][t] + lds[1][t]) + (lds[2][t] + lds[3][t]);
    }
}

// The same, finished as the forward pass is (a short, deep product).
template <typename T>
__global__ void __launch_bounds__(256)
join_forward(const GemmParams p, const float* __restrict__ parts)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, count = p.rows * p.outs;
    if (i >= count) return;
    const int64_t row = i / p.outs, out = i - row * p.outs;
    float y[1] = {0.f};
    for (int32_t k = 0; k < p.splits; ++k) y[0] += parts[k * count + i];
    if (p.bias) y[0] += (float)reinterpret_cast<const T*>(p.bias)[out];
    act_values(p.act, y);
    if (p.R) y[0] += (float)reinterpret_cast<const T*>(p.R)[row * p.ldr + out];
    reinterpret_cast<T*>(p.C)[i] = (T)y[0];
}

template <typename T>
__global__ void __launch_bounds__(256)
fill_zero(T* __restrict__ out, int64_t count)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = (T)0.f;
}

__global__ void warm_gemm_kernel() {}

hipError_t warm_gemm(hipStream_t s)
{
    hipLaunchKernelGGL(warm_gemm_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------ launches

constexpr int64_t kFewRows = 64, kManyRows = 48 * 1024;
constexpr int64_t kSumShares = 64, kSumRows = 512;

// Many rows of few inputs (rows_kernel; W's columns of a workgroup are no fewer than
// 192, and the rows are read once for each so many).  Microseconds so and by tiles,
// no activation, M of 384 to 4,096: 50,000 x 128 -> 384 15 and 20; 100,000 x 256 ->
// 4,096 304 and 370; 100,000 x 32 -> 4,096 183 and 232; 500,000 x 128 -> 512 136 and
// 227; but 20,000 x 128 -> 384 13 and 10, 20,000 x 256 -> 256 11.3 and 10.8.  With
// gelu's slope and its sums: 50,000 x 128 -> 384 38 and 45, 100,000 x 256 -> 4,096 579
// and 805, 500,000 x 128 -> 512 350 and 511; but 20,000 x 128 -> 384 36 and 23.
// dx (W's values one by one, once per workgroup): 200,003 x 128 -> 512 48 and 62,
// 100,000 x 256 -> 4,096 327 and 360; but 65,536 x 256 -> 512 37 and 30.
static bool takes_rows(const GemmParams& p)
{
    return p.rows >= (p.q_steps ? 2 : 1) * kManyRows && p.depth <= 256 && p.outs % 32 == 0 &&
           p.outs <= 8192 && way_of(p, false, p.q_steps) == kWhole;
}

template <typename T, int KF, int MODE>
static void launch_rows(GemmParams p, int32_t cus, int64_t* workgroups, hipStream_t st)
{
    constexpr int64_t most = rows_cols(KF, MODE) / 32 * 32;
    const int64_t ny = ceil_div(p.outs, most);
    const int64_t unit = p.outs % 64 == 0 && most % 64 == 0 ? 64 : 32;   // whole lines where M allows
    p.split = ceil_div(ceil_div(p.outs, ny), unit) * unit;
    const int64_t need = ceil_div(ceil_div(p.rows, 16), kRowWaves);
    *workgroups = std::max<int64_t>(1, std::min<int64_t>(need, cus / ny));
    hipLaunchKernelGGL((rows_kernel<T, KF, MODE>), dim3((unsigned)*workgroups, (unsigned)ny),
                       dim3(kRowWaves * kWave), 0, st, p);
}

template <typename T>
static f3s_status many_rows(const GemmParams& p, bool slope, int64_t* workgroups, hipStream_t st)
{
    int dev = 0, cus = 0;
    F3S_HIP(hipGetDevice(&dev));
    F3S_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    auto go = [&](auto kf) {
        constexpr int KF = decltype(kf)::value;
        if (slope) launch_rows<T, KF, kRowsSlope>(p, cus, workgroups, st);
        else if (p.R) launch_rows<T, KF, kRowsResidual>(p, cus, workgroups, st);
        else launch_rows<T, KF, kRowsAct>(p, cus, workgroups, st);
    };
    if (p.depth <= 64) go(std::integral_constant<int, 2>{});
    else if (p.depth <= 128) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

template <typename T>
static f3s_status forward(GemmParams p, void* ws, hipStream_t st)
{
    if (takes_rows(p)) {
        int64_t workgroups;
        return many_rows<T>(p, false, &workgroups, st);
    }
    if (p.rows <= kFewRows) {
        const bool fast = ((uintptr_t)p.P & 15) == 0 && ((uintptr_t)p.Q & 15) == 0 &&
                          p.depth % 8 == 0 && p.ldp % 8 == 0;
        const dim3 grid((unsigned)ceil_div(p.outs, 16));
        auto go = [&](auto nt) {
            if (fast)
                hipLaunchKernelGGL((few_rows_kernel<T, decltype(nt)::value, true>), grid, dim3(512),
                                   0, st, p);
            else
                hipLaunchKernelGGL((few_rows_kernel<T, decltype(nt)::value, false>), grid,
                                   dim3(512), 0, st, p);
        };
        if (p.rows <= 16) go(std::integral_constant<int, 1>{});
        else if (p.rows <= 32) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 4>{});
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    const Tiling t = tiling(p.rows, p.outs, p.depth, kForwardLeast, p.depth % 8 != 0, false);
    if (t.splits == 1) return launch_gemm<T, false, false, kEpiForward>(p, t, st);
    GemmParams part = p;
    part.C = static_cast<char*>(ws);
    part.bias = part.R = nullptr;
    F3S_TRY((launch_gemm<T, false, false, kEpiPart>(part, t, st)));
    p.splits = t.splits;
    hipLaunchKernelGGL((join_forward<T>), dim3((unsigned)ceil_div(p.rows * p.outs, 256)), dim3(256),
                       0, st, p, static_cast<const float*>(ws));
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

static size_t forward_bytes(int64_t n, int64_t K, int64_t M)
{
    if (n <= kFewRows) return 0;
    const int32_t s = tiling(n, M, K, kForwardLeast, K % 8 != 0, false).splits;
    return s == 1 ? 0 : up256(sizeof(float) * (size_t)s * n * M);
}

// Workspace of a backward call: dz, the sums of its columns and their shares (act),
// the splits of the products (one after another), db's.
struct BackwardSpace {
    size_t dz = 0, sums = 0, shares = 0, parts = 0, db = 0, bytes = 0;
    Tiling slope{}, dx{}, dw{};
    int64_t sum_rows = 0;
};
static BackwardSpace backward_space(int64_t n, int64_t K, int64_t M, int32_t act)
{
    BackwardSpace s;
    const bool odd_k = K % 8 != 0, odd = odd_k || M % 8 != 0;
    s.dx = tiling(n, K, M, kForwardLeast, odd, false);
    size_t parts = s.dx.splits > 1 ? sizeof(float) * (size_t)s.dx.splits * n * K : 0;
    if (act != kActNone) {
        s.slope = tiling(n, M, K, kForwardLeast, odd_k, false);
        if (s.slope.splits > 1)
            parts = std::max(parts, sizeof(float) * (size_t)s.slope.splits * n * M);
        s.sum_rows = 2 * ceil_div(n, std::min(s.slope.tile, 64));   // (at most)
        s.dz = 0;
        s.sums = up256(2 * (size_t)n * M);
        s.shares = s.sums + up256(sizeof(float) * (size_t)s.sum_rows * M);
        s.parts = s.shares + up256(sizeof(float) * (size_t)kSumShares * M);
    }
    // dW of one split is written at once; db alone (no activation) still has a product,
    // of at most eight columns, whose sums are all that is read
    s.dw = tiling(M, K, n, kWeightLeast, odd, true, act == kActNone);
    if (s.dw.splits > 1)
        parts = std::max(parts, sizeof(float) * (size_t)s.dw.splits * M * K);
    else if (act == kActNone)
        parts = std::max(parts, sizeof(float) * (size_t)M * std::min<int64_t>(K, kDbOuts));
    s.db = s.parts + up256(parts);
    s.bytes = s.db + up256(sizeof(float) * (size_t)s.dw.splits * M);
    return s;
}

struct LinearArgs {
    const char *X, *W, *bias, *dY;
    int64_t ldx, lddy;
    char *dX, *dW, *db;
    int64_t n, K, M;
    int32_t act;
};

template <typename T>
static f3s_status join(const char* parts, int64_t count, int32_t splits, char* out, const float* sums,
                       int64_t nsums, char* db, hipStream_t st)
{
    auto go = [&](auto ways) {
        constexpr int kWays = decltype(ways)::value;
        hipLaunchKernelGGL((join_splits<T, kWays>),
                           dim3((unsigned)ceil_div(count + nsums, 256 / kWays)), dim3(256), 0, st,
                           reinterpret_cast<const float*>(parts), count, splits,
                           reinterpret_cast<T*>(out), sums, nsums, reinterpret_cast<T*>(db));
    };
    if (splits <= 8) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 4>{});
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

template <typename T>
static f3s_status backward(const LinearArgs& a, char* ws, hipStream_t st)
{
    const BackwardSpace s = backward_space(a.n, a.K, a.M, a.act);
    const char* dz = a.dY;
    int64_t lddz = a.lddy;
    bool db_left = a.db != nullptr;
    if (a.act != kActNone) {
        GemmParams p{};
        p.P = a.X;
        p.ldp = a.ldx;
        p.Q = a.W;
        p.ldq = a.K;
        p.rows = a.n;
        p.outs = a.M;
        p.depth = a.K;
        p.bias = a.bias;
        p.R = a.dY;
        p.ldr = a.lddy;
        p.C = ws + s.dz;
        p.sums = a.db ? reinterpret_cast<float*>(ws + s.sums) : nullptr;
        p.act = a.act;
        int64_t sum_rows;
        if (takes_rows(p)) {
            F3S_TRY(many_rows<T>(p, true, &sum_rows, st));
        } else if (s.slope.splits > 1) {
            GemmParams part = p;
            part.C = ws + s.parts;
            part.bias = part.R = nullptr;
            F3S_TRY((launch_gemm<T, false, false, kEpiPart>(part, s.slope, st)));
            p.splits = s.slope.splits;
            sum_rows = ceil_div(a.n, 32);
            hipLaunchKernelGGL((join_slope<T>), dim3((unsigned)ceil_div(a.M, 64), (unsigned)sum_rows),
                               dim3(256), 0, st, p, reinterpret_cast<const float*>(ws + s.parts));
            F3S_HIP(hipGetLastError());
        } else {
            sum_rows = 2 * ceil_div(a.n, tile_size(s.slope, way_of(p), kEpiSlope));
            F3S_TRY((launch_gemm<T, false, false, kEpiSlope>(p, s.slope, st)));
        }
        dz = ws + s.dz;
        lddz = a.M;
        if (db_left) {
            const float* sums = p.sums;
            const unsigned nx = (unsigned)ceil_div(a.M, 64);
            if (sum_rows > kSumRows) {   // shares of them first
                float* shares = reinterpret_cast<float*>(ws + s.shares);
                const int64_t ny = std::min<int64_t>(kSumShares, ceil_div(sum_rows, 64));
                hipLaunchKernelGGL((column_sums<float>), dim3(nx, (unsigned)ny), dim3(256), 0, st,
                                   sums, sum_rows, a.M, shares);
                sums = shares;
                sum_rows = ny;
            }
            hipLaunchKernelGGL((column_sums<T>), dim3(nx, 1), dim3(256), 0, st, sums, sum_rows, a.M,
                               reinterpret_cast<T*>(a.db));
            F3S_HIP(hipGetLastError());
            db_left = false;
        }
    }
    if (a.dX) {
        GemmParams p{};
        p.P = dz;
        p.ldp = lddz;
        p.Q = a.W;
        p.ldq = a.K;
        p.rows = a.n;
        p.outs = a.K;
        p.depth = a.M;
        p.C = a.dX;
        p.q_steps = true;
        int64_t workgroups;
        if (takes_rows(p)) {
            F3S_TRY(many_rows<T>(p, false, &workgroups, st));
        } else if (s.dx.splits == 1) {
            F3S_TRY((launch_gemm<T, false, true, kEpiPlain>(p, s.dx, st)));
        } else {
            p.C = ws + s.parts;
            F3S_TRY((launch_gemm<T, false, true, kEpiPart>(p, s.dx, st)));
            F3S_TRY((join<T>(ws + s.parts, a.n * a.K, s.dx.splits, a.dX, nullptr, 0, nullptr, st)));
        }
    }
    if (a.dW || db_left) {
        GemmParams p{};
        p.P = dz;
        p.ldp = lddz;
        p.Q = a.X;
        p.ldq = a.ldx;
        p.rows = a.M;
        p.outs = a.dW ? a.K : std::min<int64_t>(a.K, kDbOuts);   // (db alone: one column of tiles)
        p.depth = a.n;
        p.sums = db_left ? reinterpret_cast<float*>(ws + s.db) : nullptr;
        // (one split: no sums to join; 4,096 x 4,096 of 4,096 rows 145 us, 181 with them)
        const bool whole = a.dW && s.dw.splits == 1;
        p.C = whole ? a.dW : ws + s.parts;
        if (whole && p.sums) F3S_TRY((launch_gemm<T, true, true, kEpiPlainSums>(p, s.dw, st)));
        else if (whole) F3S_TRY((launch_gemm<T, true, true, kEpiPlain>(p, s.dw, st)));
        else if (p.sums) F3S_TRY((launch_gemm<T, true, true, kEpiPartSums>(p, s.dw, st)));
        else F3S_TRY((launch_gemm<T, true, true, kEpiPart>(p, s.dw, st)));
        const int64_t count = a.dW && !whole ? a.M * a.K : 0, nsums = db_left ? a.M : 0;
        if (count + nsums > 0)
            F3S_TRY((join<T>(ws + s.parts, count, s.dw.splits, a.dW, p.sums, nsums, a.db, st)));
    }
    return F3S_OK;
}

static f3s_status check_linear(int64_t n, int64_t K, int64_t M, int32_t act, int32_t dtype,
                               const char* who)
{
    if (n < 0 || K < 1 || M < 1 || act < kActNone || act > kActSilu ||
        (dtype != F3S_F16 && dtype != F3S_BF16)) {
        set_error(std::string(who) + ": bad size, activation or dtype");
        return F3S_EINVAL;
    }
    if (K >= (1 << 22) || M >= (1 << 22) || n >= ((int64_t)1 << 36)) {
        set_error(std::string(who) + ": K and M below 2^22, n below 2^36");
        return F3S_EUNSUPPORTED;
    }
    return F3S_OK;
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_linear_workspace(int64_t n, int64_t K, int64_t M, int32_t act, int32_t backward_pass,
                                int64_t* bytes)
{
    F3S_REQUIRE(bytes, "f3s_linear_workspace: NULL pointer");
    F3S_TRY(check_linear(n, K, M, act, F3S_F16, "f3s_linear_workspace"));
    *bytes = (int64_t)(n == 0 ? 0 : backward_pass ? backward_space(n, K, M, act).bytes
                                                  : forward_bytes(n, K, M));
    return F3S_OK;
}

f3s_status f3s_linear_tiling(int64_t n, int64_t K, int64_t M, int32_t act, int32_t bias,
                             int32_t product, int32_t* kernel, int32_t* tile, int32_t* splits,
                             int64_t* tiles, int64_t* workgroups, int32_t* pieces)
{
    F3S_TRY(check_linear(n, K, M, act, F3S_F16, "f3s_linear_tiling"));
    F3S_REQUIRE(n > 0 && product >= F3S_LINEAR_FORWARD && product <= F3S_LINEAR_DW,
                "f3s_linear_tiling: no rows, or an unknown product");
    const char* aligned = reinterpret_cast<const char*>((uintptr_t)256);
    const BackwardSpace s = backward_space(n, K, M, act);
    const bool dx = product == F3S_LINEAR_DX, dw = product == F3S_LINEAR_DW;
    const bool sums = dw && bias && act == kActNone;   // db beside dW
    GemmParams p{};
    p.P = p.Q = aligned;
    p.C = const_cast<char*>(aligned);
    p.rows = dw ? M : n;
    p.outs = dx || dw ? K : M;
    p.depth = dx ? M : dw ? n : K;
    p.ldp = dx || dw ? M : K;
    p.ldq = K;
    p.q_steps = dx;
    if (product == F3S_LINEAR_SLOPE) {
        p.R = aligned;
        p.ldr = M;
    }
    const Tiling t = dx ? s.dx : dw ? s.dw
                                    : tiling(n, M, K, kForwardLeast, K % 8 != 0, false);
    const Way way = way_of(p, dw, dx || dw);
    const bool parts = t.splits > 1;
    const int epi = dw ? (sums ? (parts ? kEpiPartSums : kEpiPlainSums)
                               : parts ? kEpiPart : kEpiPlain)
                       : parts ? kEpiPart
                               : dx ? kEpiPlain
                                    : product == F3S_LINEAR_SLOPE ? kEpiSlope : kEpiForward;
    const int32_t kind = !dw && takes_rows(p) ? F3S_LINEAR_W_IN_LDS
                         : product == F3S_LINEAR_FORWARD && n <= kFewRows ? F3S_LINEAR_FEW_ROWS
                                                                          : F3S_LINEAR_TILES;
    const bool tiled = kind == F3S_LINEAR_TILES;
    const int32_t size = tiled ? tile_size(t, way, epi) : 0;
    const int64_t count = tiled ? ceil_div(p.rows, size) * ceil_div(p.outs, size) : 0;
    if (kernel) *kernel = kind;
    if (tile) *tile = size;
    if (splits) *splits = tiled ? t.splits : 1;
    if (tiles) *tiles = count;
    if (workgroups) *workgroups = tiled ? workgroups_of(count, size, t.splits) : 0;
    if (pieces) *pieces = way;
    return F3S_OK;
}

f3s_status f3s_linear_fwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                          const uint16_t* bias, const uint16_t* R, int64_t r_stride, uint16_t* Y,
                          int64_t n, int64_t K, int64_t M, int32_t act, int32_t dtype,
                          void* workspace, int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_linear(n, K, M, act, dtype, "f3s_linear_fwd"));
    if (n == 0) return F3S_OK;
    F3S_REQUIRE(X && W && Y, "f3s_linear_fwd: NULL pointer");
    F3S_REQUIRE(x_stride >= K && (!R || r_stride >= M), "f3s_linear_fwd: row strides below K or M");
    F3S_REQUIRE(workspace_bytes >= (int64_t)forward_bytes(n, K, M) &&
                    (workspace || workspace_bytes == 0) && ((uintptr_t)workspace & 15) == 0,
                "f3s_linear_fwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    GemmParams p{};
    p.P = reinterpret_cast<const char*>(X);
    p.ldp = x_stride;
    p.Q = reinterpret_cast<const char*>(W);
    p.ldq = K;
    p.rows = n;
    p.outs = M;
    p.depth = K;
    p.bias = reinterpret_cast<const char*>(bias);
    p.R = reinterpret_cast<const char*>(R);
    p.ldr = r_stride;
    p.C = reinterpret_cast<char*>(Y);
    p.act = act;
    if (dtype == F3S_F16) return forward<_Float16>(p, workspace, as_stream(stream));
    return forward<__bf16>(p, workspace, as_stream(stream));
}

f3s_status f3s_linear_bwd(const uint16_t* X, int64_t x_stride, const uint16_t* W,
                          const uint16_t* bias, const uint16_t* dY, int64_t dy_stride, uint16_t* dX,
                          uint16_t* dW, uint16_t* db, int64_t n, int64_t K, int64_t M, int32_t act,
                          int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_linear(n, K, M, act, dtype, "f3s_linear_bwd"));
    F3S_REQUIRE(n == 0 || (X && W && dY), "f3s_linear_bwd: NULL pointer");
    F3S_REQUIRE(n == 0 || (x_stride >= K && dy_stride >= M),
                "f3s_linear_bwd: row strides below K or M");
    F3S_REQUIRE(n == 0 || (workspace_bytes >= (int64_t)backward_space(n, K, M, act).bytes &&
                           workspace && ((uintptr_t)workspace & 15) == 0),
                "f3s_linear_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    if (n == 0) {
        auto zero = [&](uint16_t* out, int64_t count) {
            if (out)
                // (below a grid's limit of threads)
                hipLaunchKernelGGL((fill_zero<_Float16>),
                                   dim3((unsigned)std::min<int64_t>(ceil_div(count, 256), 1 << 20)),
                                   dim3(256), 0, st, reinterpret_cast<_Float16*>(out), count);
        };
        zero(dW, M * K);
        zero(db, M);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    const LinearArgs a{reinterpret_cast<const char*>(X), reinterpret_cast<const char*>(W),
                       reinterpret_cast<const char*>(bias), reinterpret_cast<const char*>(dY),
                       x_stride, dy_stride, reinterpret_cast<char*>(dX),
                       reinterpret_cast<char*>(dW), reinterpret_cast<char*>(db), n, K, M, act};
    if (dtype == F3S_F16) return backward<_Float16>(a, static_cast<char*>(workspace), st);
    return backward<__bf16>(a, static_cast<char*>(workspace), st);
}

}  // extern "C"
