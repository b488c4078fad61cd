// gemm.hip -- y = act(x W^T + b) + r and its gradient, any sizes, binary16 and
// bfloat16 with float32 sums.
//
// One tiled product serves all three directions: C[row][out] = sum_c P(row, c)
// Q(out, c), where an operand lies row by row ([row][c]) or contraction by
// contraction ([c][row]):
//   forward  P = x [n][K],      Q = W [M][K]
//   dz       the same again, dz = dy act'(z) in its epilogue: z is not kept from
//            the forward pass (n M values of memory and their traffic; in 16 bits
//            its rounding would double dz's)
//   dx       P = dz [n][M],     Q = W, transposed
//   dW       P, Q = dz, x, both transposed, n cut into splits whose float32
//            sums are added in order; db with it
// A workgroup of four waves owns a TILE x TILE block of C, 64 contraction steps
// at a time: both operands' tiles go from memory straight into LDS (16 bytes a
// lane, no registers), one ahead of the products, in an order in which neither
// plain nor transposing LDS reads meet bank conflicts.  Q is the MFMA's A operand,
// so a lane holds four consecutive outputs of a row; the epilogue passes them
// through LDS, 16 rows at a time, so that whole lines are read (residual, dy) and
// written.
#include <algorithm>

#include "half_types.hpp"

namespace f3s {

enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };
enum Epilogue : int {
    kEpiForward = 0,   // act(z + bias) + residual
    kEpiSlope = 1,     // dy act'(z + bias), and the sums of its columns
    kEpiPlain = 2,     // z
    kEpiPart = 3,      // z in float32, one slice per split
};

struct GemmParams {
    const char* P;        // operands and results: 16-bit values unless said otherwise
    const char* Q;
    int64_t ldp, ldq;     // values between rows as stored
    int64_t rows, outs, depth;
    const char* bias;     // [outs] or NULL
    const char* R;        // residual (forward, NULL: none) or dy (slope)
    int64_t ldr;
    char* C;              // [rows][outs]
    float* sums;          // slope: [row tiles][2][outs]; splits of dW: [splits][rows], NULL: none
    int64_t split;        // contraction steps per split (a multiple of 64)
    int32_t act;
    int32_t row_tiles, out_tiles, splits;
};

// erf by Abramowitz and Stegun 7.1.26 (absolute error 1.5e-7), here of z / sqrt 2
// as the normal distribution's Phi(z), with e = exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float& e)
{
    const float a = __builtin_fabsf(z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, a, 1.f));
    e = fast_exp2(-0.72134752f * z * z);   // log2(e) / 2
    float s = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    s = __builtin_fmaf(s, t, 1.421413741f);
    s = __builtin_fmaf(s, t, -0.284496736f);
    s = __builtin_fmaf(s, t, 0.254829592f);
    const float tail = 0.5f * s * t * e;   // Phi(-|z|)
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float logistic(float z)
{
    return __builtin_amdgcn_rcpf(1.f + fast_exp2(-1.44269504f * z));
}
constexpr float kTanhA = 0.79788456f, kTanhB = 0.044715f;   // sqrt(2 / pi)

__device__ __forceinline__ float act_value(int act, float z)
{
    float e;
    switch (act) {
    case kActRelu: return z < 0.f ? 0.f : z;   // (NaN stays)
    case kActGelu: return z * normal_cdf(z, e);
    case kActGeluTanh: return z * logistic(2.f * kTanhA * z * __builtin_fmaf(kTanhB * z, z, 1.f));
    case kActSilu: return z * logistic(z);
    default: return z;
    }
}
__device__ __forceinline__ float act_slope(int act, float z)
{
    float e;
    switch (act) {
    case kActRelu: return z > 0.f ? 1.f : z == z ? 0.f : z;
    case kActGelu: {
        const float c = normal_cdf(z, e);
        return __builtin_fmaf(0.39894228f * z, e, c);   // 1 / sqrt(2 pi)
    }
    case kActGeluTanh: {   // (1 + tanh u) / 2 is the logistic function of 2 u
        const float s = logistic(2.f * kTanhA * z * __builtin_fmaf(kTanhB * z, z, 1.f));
        return s + z * s * (1.f - s) * 2.f * kTanhA * __builtin_fmaf(3.f * kTanhB * z, z, 1.f);
    }
    case kActSilu: {
        const float s = logistic(z);
        return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
    }
}

// Where piece p (16 bytes) of a stored row lies in LDS, by exclusive or.  Row by
// row: 128-byte rows, whose piece of one number 16 rows' lanes read together.
__device__ __forceinline__ int place_rows(int row) { return (row >> 1) & 7; }
// Contraction by contraction: the transposing reads take rows 8 g + i, i < 4,
// and pairs of pieces, two groups g at once.
template <int TILE>
__device__ __forceinline__ int place_steps(int row)
{
    if constexpr (TILE == 128)
        return ((row & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 2) & 1);
    else
        return (row & 2) | (((row >> 3) & 1) << 2);
}

constexpr int kStep = 64;   // contraction steps per tile

// Loads one operand's tile, rows (or outputs) from `first` and steps from `step`,
// into LDS at `lds`.  FAST: rows 16-byte aligned, whole pieces inside or outside.
template <typename T, bool TRANS, int TILE, bool FAST>
__device__ __forceinline__ void load_tile(const char* base, int64_t ld, int64_t first, int64_t count,
                                          int64_t step, int64_t end, char* lds, int wave, int lane)
{
    constexpr int kPieces = (TRANS ? TILE : kStep) / 8;     // per stored row
    constexpr int kLoads = TILE * kStep * 2 / 1024 / 4;     // 1,024 bytes per wave and load
    // stored rows and columns from here on
    const int64_t r0 = TRANS ? step : first, c0 = TRANS ? first : step;
    const int64_t rows = (TRANS ? end : count) - r0, cols = (TRANS ? count : end) - c0;
    const char* src = base + (r0 * ld + c0) * 2;
    const int row_in = lane / kPieces, pos = lane % kPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int chunk = i * 4 + wave;
        const int row = chunk * (64 / kPieces) + row_in;
        const int piece = pos ^ (TRANS ? place_steps<TILE>(row) : place_rows(row));
        char* to = lds + chunk * 1024;
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(src, 0x7fffffffu);
            const bool in = row < rows && piece * 8 < cols;
            const uint32_t at = in ? (uint32_t)(row * (int32_t)ld + piece * 8) * 2 : 0xffffff00u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rs, (__attribute__((address_space(3))) void*)to, 16, (int)at, 0, 0, 0);
        } else {
            typename Half<T>::v8 v = {};
            const T* p = reinterpret_cast<const T*>(src) + row * ld + piece * 8;
            if (row < rows) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (piece * 8 + k < cols) v[k] = p[k];
            }
            *reinterpret_cast<typename Half<T>::v8*>(to + lane * 16) = v;
        }
    }
}

// Operand fragment: 16 rows from 16 t, contraction 32 f + 8 g ..
template <typename T, bool TRANS, int TILE>
__device__ __forceinline__ typename Half<T>::v8 fragment(const char* lds, int t, int f, int lane)
{
    const int g = lane >> 4, r = lane & 15;
    if constexpr (!TRANS) {
        return *reinterpret_cast<const typename Half<T>::v8*>(
            lds + (16 * t + r) * 128 + 16 * ((4 * f + g) ^ place_rows(r)));
    } else {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4* lds4;
        // lane r hands out piece part r % 4 of row r / 4 and receives column r
        const int i = r >> 2, c = r & 3;
        s4 h[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = 32 * f + 8 * g + 4 * u + i;
            const char* at = lds + row * (TILE * 2) +
                             16 * ((2 * t + (c >> 1)) ^ place_steps<TILE>(row)) + 8 * (c & 1);
            h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
        }
        return __builtin_bit_cast(typename Half<T>::v8, s8{h[0][0], h[0][1], h[0][2], h[0][3],
                                                           h[1][0], h[1][1], h[1][2], h[1][3]});
    }
}

// Workgroup -> tile.  Each XCD takes a contiguous range of them (the dispatcher
// deals workgroups to the XCDs in turn), in groups of 8 row tiles by all output
// tiles: the row tiles' operand stays in its L2 while the others pass by.
__device__ __forceinline__ void tile_of(const GemmParams& p, int32_t& row, int32_t& out)
{
    const int64_t G = (int64_t)p.row_tiles * p.out_tiles, b = blockIdx.x;
    const int64_t x = b % kXcds, q = G / kXcds, rem = G % kXcds;
    const int64_t id = x * q + min(x, rem) + b / kXcds;
    constexpr int kGroup = 8;
    const int64_t group = id / ((int64_t)kGroup * p.out_tiles);
    const int64_t first = group * kGroup, in = id - first * p.out_tiles;
    const int64_t size = min((int64_t)kGroup, (int64_t)p.row_tiles - first);
    row = (int32_t)(first + in % size);
    out = (int32_t)(in / size);
}

// Eight values at C's (row, out ..) from float32: bias, activation, residual, rounding.
template <typename T, int EPI, bool FAST>
__device__ __forceinline__ void finish8(const GemmParams& p, int64_t row, int64_t out, f4 lo, f4 hi,
                                        float (&sum)[8])
{
    typedef typename Half<T>::v8 v8;
    float z[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    const int64_t left = p.outs - out;
    if (row >= p.rows || left <= 0) return;
    const int many = FAST ? 8 : (int)min((int64_t)8, left);   // (FAST: outs % 8 == 0)
    auto load = [&](const T* src, float (&x)[8]) __attribute__((always_inline)) {
        if constexpr (FAST) {
            const v8 v = *reinterpret_cast<const v8*>(src);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (float)v[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = k < many ? (float)src[k] : 0.f;
        }
    };
    if constexpr (EPI == kEpiForward || EPI == kEpiSlope) {
        if (p.bias) {
            float b[8];
            load(reinterpret_cast<const T*>(p.bias) + out, b);
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] += b[k];
        }
        float r[8] = {};
        if (p.R) load(reinterpret_cast<const T*>(p.R) + row * p.ldr + out, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if constexpr (EPI == kEpiForward) {
                z[k] = act_value(p.act, z[k]) + r[k];
            } else {
                z[k] = r[k] * act_slope(p.act, z[k]);
                sum[k] += z[k];
            }
        }
    }
    T* dst = reinterpret_cast<T*>(p.C) + row * p.outs + out;
    if constexpr (FAST) {
        typedef float f8 __attribute__((ext_vector_type(8)));
        *reinterpret_cast<v8*>(dst) = __builtin_convertvector(
            (f8{z[0], z[1], z[2], z[3], z[4], z[5], z[6], z[7]}), v8);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < many) dst[k] = (T)z[k];
    }
}

template <typename T, bool PT, bool QT, int TILE, int EPI, bool FAST>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
gemm_kernel(const GemmParams p)
{
    typedef typename Half<T>::v8 v8;
    constexpr int kTileBytes = TILE * kStep * 2;
    constexpr int kW = TILE / 2;         // a wave's block of C is kW x kW
    constexpr int kN = kW / 16;
    constexpr int kOutRow = kW + 4;      // floats of a staged row
    __shared__ __align__(256) char lds[2][2][kTileBytes];   // [buffer][P, Q]
    static_assert(sizeof(lds) >= 4 * 16 * kOutRow * sizeof(float), "the waves' epilogue stages");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int wr = wave >> 1, wo = wave & 1;
    int32_t rt, ot;
    tile_of(p, rt, ot);
    const int64_t row0 = (int64_t)rt * TILE, out0 = (int64_t)ot * TILE;
    const int64_t begin = (int64_t)blockIdx.y * p.split, end = min(p.depth, begin + p.split);

    f4 acc[kN][kN];   // [outputs][rows]
    f4 col[kN];       // sums of P's rows (dW's splits: db)
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        col[i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kN; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    const bool with_sums = EPI == kEpiPart && p.sums && ot == 0 && wo == 0;
    v8 ones;
#pragma unroll
    for (int k = 0; k < 8; ++k) ones[k] = (T)1.f;

    auto load = [&](int64_t c, int buf) __attribute__((always_inline)) {
        load_tile<T, PT, TILE, FAST>(p.P, p.ldp, row0, p.rows, c, end, lds[buf][0], wave, lane);
        load_tile<T, QT, TILE, FAST>(p.Q, p.ldq, out0, p.outs, c, end, lds[buf][1], wave, lane);
    };
    if (begin < end) load(begin, 0);
    int buf = 0;
    for (int64_t c = begin; c < end; c += kStep, buf ^= 1) {
        // this tile has landed (loads into LDS are waited for by hand: the barrier
        // does not), and the last one's readers are done
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        __syncthreads();
        if (c + kStep < end) load(c + kStep, buf ^ 1);
        const char* pt = lds[buf][0];
        const char* qt = lds[buf][1];
#pragma unroll
        for (int f = 0; f < kStep / 32; ++f) {
            v8 a[kN], b[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                a[i] = fragment<T, QT, TILE>(qt, kN * wo + i, f, lane);
                b[i] = fragment<T, PT, TILE>(pt, kN * wr + i, f, lane);
            }
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int j = 0; j < kN; ++j) acc[i][j] = Half<T>::mfma(a[i], b[j], acc[i][j]);
            if (with_sums) {
#pragma unroll
                for (int j = 0; j < kN; ++j) col[j] = Half<T>::mfma(ones, b[j], col[j]);
            }
        }
    }
    __syncthreads();

    float* stage = reinterpret_cast<float*>(&lds[0][0][0]) + wave * 16 * kOutRow;
    float sum[8] = {};
    constexpr int kLanes = kW / 8;           // lanes per row of the block, 8 outputs each
    constexpr int kRowsAtOnce = kWave / kLanes;
    const int64_t out = out0 + kW * wo + 8 * (lane % kLanes);
    float* part = EPI == kEpiPart ? reinterpret_cast<float*>(p.C) +
                                        (int64_t)blockIdx.y * p.rows * p.outs : nullptr;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < kN; ++i)
            *reinterpret_cast<f4*>(&stage[r * kOutRow + 16 * i + 4 * g]) = acc[i][j];
        wave_lds_order();
#pragma unroll
        for (int v = 0; v < 16 / kRowsAtOnce; ++v) {
            const int rr = v * kRowsAtOnce + lane / kLanes;
            const float* src = &stage[rr * kOutRow + 8 * (lane % kLanes)];
            const f4 lo = *reinterpret_cast<const f4*>(src), hi = *reinterpret_cast<const f4*>(src + 4);
            const int64_t row = row0 + kW * wr + 16 * j + rr;
            if constexpr (EPI == kEpiPart) {
                if (row < p.rows && out < p.outs) {
                    float* dst = part + row * p.outs + out;
                    if constexpr (FAST) {
                        *reinterpret_cast<f4*>(dst) = lo;
                        *reinterpret_cast<f4*>(dst + 4) = hi;
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (out + k < p.outs) dst[k] = k < 4 ? lo[k & 3] : hi[k & 3];
                    }
                }
            } else {
                finish8<T, EPI, FAST>(p, row, out, lo, hi, sum);
            }
        }
    }
    if constexpr (EPI == kEpiSlope) {
        if (p.sums) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int off = kLanes; off < kWave; off <<= 1) sum[k] += __shfl_xor(sum[k], off, kWave);
                if (lane < kLanes && out + k < p.outs)
                    p.sums[((int64_t)rt * 2 + wr) * p.outs + out + k] = sum[k];
            }
        }
    }
    if constexpr (EPI == kEpiPart) {
        if (with_sums && g == 0) {   // (every row of the ones' product is the sums)
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const int64_t row = row0 + kW * wr + 16 * j + r;
                if (row < p.rows) p.sums[(int64_t)blockIdx.y * p.rows + row] = col[j][0];
            }
        }
    }
}

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
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int64_t out = out0 + 4 * g + v;
            if (out >= p.outs) break;
            float y = z[v];
            if (p.bias) y += (float)reinterpret_cast<const T*>(p.bias)[out];
            y = act_value(p.act, y);
            if (p.R) y += (float)reinterpret_cast<const T*>(p.R)[row * p.ldr + out];
            reinterpret_cast<T*>(p.C)[row * p.outs + out] = (T)y;
        }
    }
}

// Splits of a product added in their order; `rows x outs` values, and (db) the
// sums that came with them.
template <typename T>
__global__ void __launch_bounds__(256)
join_splits(const float* __restrict__ parts, int64_t count, int32_t splits, T* __restrict__ out,
            const float* __restrict__ sums, int64_t nsums, T* __restrict__ db)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) {
        float s = 0.f;
        for (int32_t k = 0; k < splits; ++k) s += parts[k * count + i];
        out[i] = (T)s;
    } else if (i < count + nsums) {
        float s = 0.f;
        for (int32_t k = 0; k < splits; ++k) s += sums[k * nsums + i - count];
        db[i - count] = (T)s;
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
    float y = 0.f;
    for (int32_t k = 0; k < p.splits; ++k) y += parts[k * count + i];
    if (p.bias) y += (float)reinterpret_cast<const T*>(p.bias)[out];
    y = act_value(p.act, y);
    if (p.R) y += (float)reinterpret_cast<const T*>(p.R)[row * p.ldr + out];
    reinterpret_cast<T*>(p.C)[i] = (T)y;
}

// Sums of the columns of in[rows][cols]: blockIdx.y's share of the rows, 64 columns
// per workgroup, in a fixed order.  OUT: float (a share each) or the type (all).
template <typename OUT>
__global__ void __launch_bounds__(256)
column_sums(const float* __restrict__ in, int64_t rows, int64_t cols, OUT* __restrict__ out)
{
    __shared__ float lds[4][64];
    const int64_t col = (int64_t)blockIdx.x * 64 + threadIdx.x % 64;
    const int part = threadIdx.x / 64;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    float s = 0.f;
    if (col < cols)
        for (int64_t i = r0 + part; i < r1; i += 4) s += in[i * cols + col];
    lds[part][threadIdx.x % 64] = s;
    __syncthreads();
    if (part == 0 && col < cols) {
        const int t = threadIdx.x;
        out[blockIdx.y * cols + col] = (OUT)((lds[0][t] + lds[1][t]) + (lds[2][t] + lds[3][t]));
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
fill_zero(T* __restrict__ out, int64_t count)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) out[i] = (T)0.f;
}

__global__ void warm_gemm_kernel() {}

hipError_t warm_gemm(hipStream_t s)
{
    hipLaunchKernelGGL(warm_gemm_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------ launches

constexpr int64_t kFewRows = 64;
constexpr int32_t kManyTiles = 512;   // two workgroups per CU
constexpr int64_t kSumShares = 64;

// 128 x 128 tiles where they are enough for the chip's 256 CUs, else 64 x 64.
static bool small_tiles(int64_t rows, int64_t outs)
{
    return ceil_div(rows, 128) * ceil_div(outs, 128) < 256;
}
static int64_t tiles(int64_t rows, int64_t outs, bool small)
{
    const int64_t t = small ? 64 : 128;
    return ceil_div(rows, t) * ceil_div(outs, t);
}
// Splits of a contraction of `depth` steps: as many as give every CU two
// workgroups, of `least` steps or more.
static int32_t splits_for(int64_t rows, int64_t outs, int64_t depth, int64_t least)
{
    const int64_t t = tiles(rows, outs, small_tiles(rows, outs));
    const int64_t want = std::min(ceil_div(kManyTiles, std::max<int64_t>(t, 1)), depth / least);
    return (int32_t)std::max<int64_t>(1, std::min<int64_t>(want, 256));
}
constexpr int64_t kForwardLeast = 512, kWeightLeast = 256;

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T, bool PT, bool QT, int EPI, bool FAST>
static void launch_tiles(GemmParams p, hipStream_t st)
{
    const bool small = small_tiles(p.rows, p.outs);
    const int64_t t = small ? 64 : 128;
    p.row_tiles = (int32_t)ceil_div(p.rows, t);
    p.out_tiles = (int32_t)ceil_div(p.outs, t);
    p.split = ceil_div(ceil_div(p.depth, p.splits), kStep) * kStep;
    const dim3 grid((unsigned)((int64_t)p.row_tiles * p.out_tiles), (unsigned)p.splits);
    if (small)
        hipLaunchKernelGGL((gemm_kernel<T, PT, QT, 64, EPI, FAST>), grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((gemm_kernel<T, PT, QT, 128, EPI, FAST>), grid, dim3(256), 0, st, p);
}

// FAST: whole 16-byte pieces everywhere, offsets in a tile within 31 bits.
template <typename T, bool PT, bool QT, int EPI>
static f3s_status launch_gemm(const GemmParams& p, hipStream_t st)
{
    auto rows_ok = [](const char* x, int64_t ld) {
        return ((uintptr_t)x & 15) == 0 && ld % 8 == 0 && ld < (1 << 22);
    };
    const int64_t pcols = PT ? p.rows : p.depth, qcols = QT ? p.outs : p.depth;
    const bool fast = rows_ok(p.P, p.ldp) && rows_ok(p.Q, p.ldq) && pcols % 8 == 0 &&
                      qcols % 8 == 0 && p.outs % 8 == 0 && ((uintptr_t)p.C & 15) == 0 &&
                      (!p.bias || ((uintptr_t)p.bias & 15) == 0) &&
                      (!p.R || rows_ok(p.R, p.ldr));
    if (tiles(p.rows, p.outs, small_tiles(p.rows, p.outs)) >= ((int64_t)1 << 31)) {
        set_error("linear: too many tiles");
        return F3S_EUNSUPPORTED;
    }
    if (fast) launch_tiles<T, PT, QT, EPI, true>(p, st);
    else launch_tiles<T, PT, QT, EPI, false>(p, st);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

template <typename T>
static f3s_status forward(GemmParams p, void* ws, hipStream_t st)
{
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
    p.splits = splits_for(p.rows, p.outs, p.depth, kForwardLeast);
    if (p.splits == 1) return launch_gemm<T, false, false, kEpiForward>(p, st);
    GemmParams part = p;
    part.C = static_cast<char*>(ws);
    part.bias = part.R = nullptr;
    F3S_TRY((launch_gemm<T, false, false, kEpiPart>(part, st)));
    hipLaunchKernelGGL((join_forward<T>), dim3((unsigned)ceil_div(p.rows * p.outs, 256)), dim3(256),
                       0, st, p, static_cast<const float*>(ws));
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

static size_t forward_bytes(int64_t n, int64_t K, int64_t M)
{
    if (n <= kFewRows) return 0;
    const int32_t s = splits_for(n, M, K, kForwardLeast);
    return s == 1 ? 0 : up256(sizeof(float) * (size_t)s * n * M);
}

// Workspace of a backward call: dz, the sums of its columns (act), dW's splits,
// db's.
struct BackwardSpace {
    size_t dz = 0, sums = 0, shares = 0, parts = 0, db = 0, bytes = 0;
    int32_t splits = 1;
    int64_t sum_rows = 0;
};
static BackwardSpace backward_space(int64_t n, int64_t K, int64_t M, int32_t act)
{
    BackwardSpace s;
    if (act != kActNone) {
        const int64_t t = small_tiles(n, M) ? 64 : 128;
        s.sum_rows = 2 * ceil_div(n, t);
        s.dz = 0;
        s.sums = up256(2 * (size_t)n * M);
        s.shares = s.sums + up256(sizeof(float) * (size_t)s.sum_rows * M);
        s.parts = s.shares + up256(sizeof(float) * (size_t)kSumShares * M);
    }
    s.splits = splits_for(M, K, n, kWeightLeast);
    s.db = s.parts + up256(sizeof(float) * (size_t)s.splits * M * K);
    s.bytes = s.db + up256(sizeof(float) * (size_t)s.splits * M);
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
        p.splits = 1;
        F3S_TRY((launch_gemm<T, false, false, kEpiSlope>(p, st)));
        dz = ws + s.dz;
        lddz = a.M;
        if (db_left) {
            float* shares = reinterpret_cast<float*>(ws + s.shares);
            const int64_t ny = std::min<int64_t>(kSumShares, s.sum_rows);
            const unsigned nx = (unsigned)ceil_div(a.M, 64);
            hipLaunchKernelGGL((column_sums<float>), dim3(nx, (unsigned)ny), dim3(256), 0, st,
                               p.sums, s.sum_rows, a.M, shares);
            hipLaunchKernelGGL((column_sums<T>), dim3(nx, 1), dim3(256), 0, st, shares, ny, a.M,
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
        p.splits = 1;
        F3S_TRY((launch_gemm<T, false, true, kEpiPlain>(p, st)));
    }
    if (a.dW || db_left) {
        GemmParams p{};
        p.P = dz;
        p.ldp = lddz;
        p.Q = a.X;
        p.ldq = a.ldx;
        p.rows = a.M;
        p.outs = a.K;
        p.depth = a.n;
        p.C = ws + s.parts;
        p.sums = db_left ? reinterpret_cast<float*>(ws + s.db) : nullptr;
        p.splits = s.splits;
        F3S_TRY((launch_gemm<T, true, true, kEpiPart>(p, st)));
        const int64_t count = a.dW ? a.M * a.K : 0, nsums = db_left ? a.M : 0;
        hipLaunchKernelGGL((join_splits<T>), dim3((unsigned)ceil_div(count + nsums, 256)), dim3(256),
                           0, st, reinterpret_cast<const float*>(ws + s.parts), count, s.splits,
                           reinterpret_cast<T*>(a.dW), p.sums, nsums, reinterpret_cast<T*>(a.db));
        F3S_HIP(hipGetLastError());
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
    p.splits = 1;
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
                hipLaunchKernelGGL((fill_zero<_Float16>), dim3((unsigned)ceil_div(count, 256)),
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
