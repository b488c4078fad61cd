// gemm_tiles.hpp -- the tiled product that projections (gemm.hip) and the loss of a
// classifier (cross_entropy.hip) are made of: C[row][out] = sum_c P(row, c) Q(out, c)
// and its epilogues, the sums of splits and columns after it, the choice of tiles.
#pragma once

#include <algorithm>

#include "half_types.hpp"

namespace f3s {

enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };
enum Epilogue : int {
    kEpiForward = 0,   // act(z + bias) + residual
    kEpiSlope = 1,     // dy act'(z + bias), and the sums of its columns
    kEpiPlain = 2,     // z
    kEpiPart = 3,      // z in float32, one slice per split
    kEpiPartSums = 4,  // and the sums of P's rows (dW: db)
    kEpiPlainSums = 5, // z, and those sums
    // (the loss of a classifier; the last two with q_end)
    kEpiLse = 6,       // of z + bias, per row and block of a wave's outputs: largest, sum of exp
    kEpiProb = 7,      // dz = (softmax - 1 at the target) f, and the sums of its columns
    kEpiScaled = 8,    // z times *factor
    kEpiAdd = 9,       // as kEpiPart; with `add` onto what is there
};

// What kEpiLse and kEpiProb take beside z.
struct LossParams {
    const int64_t* target;   // [rows]
    int64_t first;           // the class of output 0
    float2* blocks;          // (kEpiLse) [blocks of outputs][rows]: largest, sum
    float* picked;           // (kEpiLse) [rows]: z + bias at the target, where there is one
    const float* lse;        // (kEpiProb) [rows]
    const float* f;          // (kEpiProb) [rows]; 0: the row does not count
    int64_t outs;            // (kEpiProb) outputs; C's columns from here on become 0
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
    float* sums;          // NULL: none; slope: [row tiles][2][outs], rows_kernel [workgroups][outs];
                          // splits of dW: [splits][rows]
    int64_t split;        // contraction steps per split (a multiple of 64)
    int32_t act;
    int32_t row_tiles, out_tiles, splits;
    bool q_steps;         // rows_kernel: Q lies contraction by contraction
    bool add;             // kEpiAdd
    int64_t q_end;        // kEpiScaled, kEpiAdd: Q has this many steps (P's others are 0)
    const float* factor;  // kEpiScaled
    LossParams loss;
};

__device__ __forceinline__ float logistic(float z)
{
    return __builtin_amdgcn_rcpf(1.f + fast_exp2(-1.44269504f * z));
}
// Phi(z), the normal distribution's: the logistic function of z P(z^2), P fitted
// (weighted minimax, degree 6, to z (Phi - its value) for |z| <= 8) to
// log(Phi / (1 - Phi)) / z, positive everywhere: z Phi to 6e-7, Phi to 2e-7, and
// both tails' ends.  One exponential and one reciprocal, eight other operations;
// by erf's usual rational form there were 15.  (Where K is small the activation
// bounds the kernel: 500,000 x 128 -> 512 is 256 M of them.)
__device__ __forceinline__ float normal_cdf(float z)
{
    constexpr float c[7] = {-2.30220720e+00f,
                            -1.04838581e-01f,
                            9.55929293e-05f,
                            1.59389413e-04f,
                            -1.14524302e-05f,
                            3.85045013e-07f,
                            -5.20990915e-09f};   // by -log2(e)
    const float t = z * z;
    float s = c[6];
#pragma unroll
    for (int k = 5; k >= 0; --k) s = __builtin_fmaf(s, t, c[k]);
    return __builtin_amdgcn_rcpf(1.f + fast_exp2(z * s));
}
constexpr float kTanhA = 0.79788456f, kTanhB = 0.044715f;   // sqrt(2 / pi)

__device__ __forceinline__ float gelu_tanh_cdf(float z)   // (1 + tanh u) / 2 = logistic(2 u)
{
    return logistic(2.f * kTanhA * z * __builtin_fmaf(kTanhB * z, z, 1.f));
}

template <int N, typename F>
__device__ __forceinline__ void each(float (&z)[N], F f)
{
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = f(z[k]);
}
// z -> act(z), and (smooth activations) z -> act'(z); act is uniform.
template <int N>
__device__ __forceinline__ void act_values(int act, float (&z)[N])
{
    switch (act) {
    case kActRelu: each(z, [](float x) { return x < 0.f ? 0.f : x; }); break;   // (NaN stays)
    case kActGelu: each(z, [](float x) { return x * normal_cdf(x); }); break;
    case kActGeluTanh: each(z, [](float x) { return x * gelu_tanh_cdf(x); }); break;
    case kActSilu: each(z, [](float x) { return x * logistic(x); }); break;
    default: break;
    }
}
template <int N>
__device__ __forceinline__ void act_slopes(int act, float (&z)[N])
{
    switch (act) {
    case kActGelu:   // Phi + x phi
        each(z, [](float x) {
            return __builtin_fmaf(0.39894228f * x, fast_exp2(-0.72134752f * x * x), normal_cdf(x));
        });
        break;
    case kActGeluTanh:
        each(z, [](float x) {
            const float s = gelu_tanh_cdf(x);
            // (s (1 - s) is 0 from |x| = 10 on; x x overflows from 2^64 on)
            const float t = __builtin_fminf(x * x, 1e4f);
            return s + x * s * (1.f - s) * 2.f * kTanhA * __builtin_fmaf(3.f * kTanhB, t, 1.f);
        });
        break;
    case kActSilu:
        each(z, [](float x) {
            const float s = logistic(x);
            return s * (1.f + x * (1.f - s));
        });
        break;
    default: each(z, [](float) { return 1.f; }); break;
    }
}
// z -> dy act'(z).  relu passes dy on or not: 0 x inf is no gradient of a unit that is off.
template <int N>
__device__ __forceinline__ void act_gradients(int act, float (&z)[N], const float (&dy)[N])
{
    if (act == kActRelu) {
#pragma unroll
        for (int k = 0; k < N; ++k) z[k] = z[k] > 0.f ? dy[k] : z[k] == z[k] ? 0.f : z[k];
        return;
    }
    act_slopes(act, z);
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] *= dy[k];
}

constexpr float kLog2eF = 1.44269504f;
constexpr int kStep = 64;   // contraction steps per tile

template <typename V>
struct __attribute__((packed, aligned(2))) Unaligned {
    V v;
};

// Where piece p (16 bytes) of a stored row lies in LDS, by exclusive or.  Row by
// row, 128 bytes each: the pieces of one number that 16 rows' lanes read together
// lie in distinct banks.
__device__ __forceinline__ int place_rows(int row) { return (row >> 1) & 7; }
// Contraction by contraction: the transposing reads take rows 8 g + i, i < 4,
// and pairs of pieces, two groups g at once.
template <int TILE>
__device__ __forceinline__ int place_steps(int row)
{
    if constexpr (TILE >= 128)
        return ((row & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 2) & 1);
    else
        return (row & 2) | (((row >> 3) & 1) << 2);
}

// One operand's tile, rows (or outputs) from `first` and steps from `step`: the
// places of its pieces.  `in` says whether piece i of a lane is (in part) inside.
template <bool TRANS, int TILE, int WAVES>
struct TileAt {
    static constexpr int pieces = (TRANS ? TILE : kStep) / 8;        // per stored row
    static constexpr int loads = TILE * kStep * 2 / 1024 / WAVES;    // 1,024 bytes per wave and load
    int64_t rows, cols;   // stored rows and columns from here on
    const char* src;
    __device__ __forceinline__ TileAt(const char* base, int64_t ld, int64_t first, int64_t count,
                                      int64_t step, int64_t end)
    {
        const int64_t r0 = TRANS ? step : first, c0 = TRANS ? first : step;
        rows = (TRANS ? end : count) - r0;
        cols = (TRANS ? count : end) - c0;
        src = base + (r0 * ld + c0) * 2;
    }
    static __device__ __forceinline__ int chunk(int i, int wave) { return i * WAVES + wave; }
    static __device__ __forceinline__ int row(int i, int wave, int lane)
    {
        return chunk(i, wave) * (64 / pieces) + lane / pieces;
    }
    static __device__ __forceinline__ int piece(int row, int lane)
    {
        return (lane % pieces) ^ (TRANS ? place_steps<TILE>(row) : place_rows(row));
    }
};

// Straight into LDS.  Rows 16-byte aligned, whole pieces inside or outside.
template <bool TRANS, int TILE, int WAVES>
__device__ __forceinline__ void load_tile(const TileAt<TRANS, TILE, WAVES>& t, int64_t ld, char* lds,
                                          int wave, int lane)
{
#pragma unroll
    for (int i = 0; i < t.loads; ++i) {
        const int row = t.row(i, wave, lane), piece = t.piece(row, lane);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(t.src, 0x7fffffffu);
        const bool in = row < t.rows && piece * 8 < t.cols;
        const uint32_t at = in ? (uint32_t)(row * (int32_t)ld + piece * 8) * 2 : 0xffffff00u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void*)(lds + t.chunk(i, wave) * 1024), 16, (int)at,
            0, 0, 0);
    }
}

// Any alignment and width: through registers, whose contents go to LDS (put_tile)
// when the products of the step before are done.  A piece that its row ends in is
// read whole where another row follows (its address stays inside then), and what is
// not the row's becomes zero.
template <typename T, bool TRANS, int TILE, int WAVES, typename V = typename Half<T>::v8>
__device__ __forceinline__ void fetch_tile(const TileAt<TRANS, TILE, WAVES>& t, int64_t ld, V* to,
                                           int wave, int lane)
{
#pragma unroll
    for (int i = 0; i < t.loads; ++i) {
        const int row = t.row(i, wave, lane), piece = t.piece(row, lane);
        const T* p = reinterpret_cast<const T*>(t.src) + row * ld + piece * 8;
        const int64_t left = row < t.rows ? t.cols - piece * 8 : 0;
        const bool whole = left >= 8 || (left > 0 && ld >= 8 && row + 1 < t.rows);
        V v = {};
        if (whole) v = reinterpret_cast<const Unaligned<V>*>(p)->v;
        if (left < 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (!whole && k < left) v[k] = p[k];
                if (k >= left) v[k] = (T)0.f;
            }
        }
        to[i] = v;
    }
}
template <bool TRANS, int TILE, int WAVES, typename V>
__device__ __forceinline__ void put_tile(const V* from, char* lds, int wave, int lane)
{
    typedef TileAt<TRANS, TILE, WAVES> At;
#pragma unroll
    for (int i = 0; i < At::loads; ++i)
        *reinterpret_cast<V*>(lds + At::chunk(i, wave) * 1024 + lane * 16) = from[i];
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

// Number -> tile.  Each XCD takes a contiguous range of them (the dispatcher deals
// workgroups to the XCDs in turn, and a workgroup's numbers are a multiple of eight
// apart), in groups of 8 row tiles by all output
// tiles: the row tiles' operand stays in its L2 while the others pass by.
__device__ __forceinline__ void tile_of(const GemmParams& p, int64_t b, int32_t& row, int32_t& out)
{
    const int64_t G = (int64_t)p.row_tiles * p.out_tiles;
    const int64_t x = b % kXcds, q = G / kXcds, rem = G % kXcds;
    const int64_t id = x * q + min(x, rem) + b / kXcds;
    constexpr int kGroup = 8;
    const int64_t group = id / ((int64_t)kGroup * p.out_tiles);
    const int64_t first = group * kGroup, in = id - first * p.out_tiles;
    const int64_t size = min((int64_t)kGroup, (int64_t)p.row_tiles - first);
    row = (int32_t)(first + in % size);
    out = (int32_t)(in / size);
}

// Eight values of an operand from `out` of `left` there are.
template <typename T, bool FAST>
__device__ __forceinline__ typename Half<T>::v8 load8(const T* src, int64_t left)
{
    typename Half<T>::v8 v = {};
    if constexpr (FAST) {   // (whole pieces)
        if (left > 0) v = *reinterpret_cast<const typename Half<T>::v8*>(src);
    } else if (left >= 8) {
        v = reinterpret_cast<const Unaligned<typename Half<T>::v8>*>(src)->v;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) v[k] = src[k];
    }
    return v;
}

// Eight values at C's (row, out ..) from float32: bias, activation, residual (or dy),
// rounding.
template <typename T, int EPI, bool FAST>
__device__ __forceinline__ void finish8(const GemmParams& p, int64_t row, int64_t out, f4 lo, f4 hi,
                                        typename Half<T>::v8 bias, typename Half<T>::v8 r,
                                        float (&sum)[8])
{
    typedef typename Half<T>::v8 v8;
    float z[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    const int64_t left = p.outs - out;
    if (row >= p.rows || left <= 0) return;
    if constexpr (EPI == kEpiScaled) {
        const float f = *p.factor;
#pragma unroll
        for (int k = 0; k < 8; ++k) z[k] *= f;
    }
    if constexpr (EPI == kEpiForward || EPI == kEpiSlope) {
#pragma unroll
        for (int k = 0; k < 8; ++k) z[k] += (float)bias[k];
        if constexpr (EPI == kEpiForward) {
            act_values(p.act, z);
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] += (float)r[k];
        } else {
            float dy[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) dy[k] = (float)r[k];
            act_gradients(p.act, z, dy);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] += z[k];
        }
    }
    T* dst = reinterpret_cast<T*>(p.C) + row * p.outs + out;
    typedef float f8 __attribute__((ext_vector_type(8)));
    const v8 y = __builtin_convertvector((f8{z[0], z[1], z[2], z[3], z[4], z[5], z[6], z[7]}), v8);
    if constexpr (FAST) {
        *reinterpret_cast<v8*>(dst) = y;
    } else if (left >= 8) {
        reinterpret_cast<Unaligned<v8>*>(dst)->v = y;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) dst[k] = y[k];
    }
}

// Tiles of C, contraction steps of 64, the next one's tiles on their way meanwhile.
// 64 and 128: a quarter for each of four waves, two workgroups per CU and more;
// 256: eight waves of 128 rows by 64 outputs.  (What bounds the small ones is the
// way from L2 to LDS, 64 bytes per clock and CU: 128 x 128 x 64 products take its
// time as long as the matrix cores'; 256 x 256 x 64 half of it.  32,768 x 1,024 ->
// 4,096, TFLOP/s: 64 560, 128 737, 256 910 and, since its second half's operands are
// read between the first half's products, 1,020; beside the 910, 256 by four waves of
// 128 x 128, a wave per SIMD, 776; three steps of 32 with the next one's operands read
// ahead into registers, 256 x 256 743, 256 x 128 698.)
template <int SIZE>
struct Shape {
    static constexpr int wave_rows = 2, wave_outs = SIZE == 256 ? 4 : 2, waves = wave_rows * wave_outs;
    static constexpr int rows = SIZE / wave_rows, outs = SIZE / wave_outs;   // of a wave
    static constexpr int tile_bytes = SIZE * kStep * 2;
};

// kWhole: whole 16-byte pieces everywhere; kTiles: of the operands' rows; kAny.
enum Way : int { kAny = 0, kTiles = 1, kWhole = 2 };
template <typename T, bool PT, bool QT, int SIZE, int EPI, int WAY>
__global__ void __launch_bounds__(Shape<SIZE>::waves * kWave) __attribute__((amdgpu_waves_per_eu(2)))
gemm_kernel(const GemmParams p)
{
    typedef typename Half<T>::v8 v8;
    typedef Shape<SIZE> S;
    constexpr bool LOADS = WAY != kAny, FAST = WAY == kWhole;   // tiles; C, bias and R
    constexpr int kNo = S::outs / 16, kNr = S::rows / 16;
    constexpr int kOutRow = S::outs + 4;      // floats of a staged row
    __shared__ __align__(256) char lds[2][2][S::tile_bytes];   // [buffer][P, Q]
    static_assert(sizeof(lds[0]) >= S::waves * 16 * kOutRow * sizeof(float), "the waves' epilogue stages");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    const int wr = wave / S::wave_outs, wo = wave % S::wave_outs;
    const int64_t begin = (int64_t)blockIdx.y * p.split, end = min(p.depth, begin + p.split);
    const int64_t total = (int64_t)p.row_tiles * p.out_tiles;
    constexpr bool kSums = EPI == kEpiPartSums || EPI == kEpiPlainSums;
    constexpr bool kPart = EPI == kEpiPart || EPI == kEpiPartSums || EPI == kEpiAdd;
    constexpr bool kLoss = EPI == kEpiLse || EPI == kEpiProb;
    constexpr bool kTail = EPI == kEpiScaled || EPI == kEpiAdd;
    // (kLoss) a tile's rows: target (-1: none here), lse, f
    struct RowInfo {
        int32_t t;
        float lse, f;
    };
    __shared__ RowInfo info[kLoss ? SIZE : 1];
    v8 ones;
    if constexpr (kSums) {
#pragma unroll
        for (int k = 0; k < 8; ++k) ones[k] = (T)1.f;
    }

    int32_t rt, ot;
    typedef TileAt<PT, SIZE, S::waves> AtP;
    typedef TileAt<QT, SIZE, S::waves> AtQ;
    v8 held_p[LOADS ? 1 : AtP::loads], held_q[LOADS ? 1 : AtQ::loads];
    // step c's tiles into buffer buf; not LOADS: on their way, put() brings them there
    auto load = [&](int64_t c, int buf) __attribute__((always_inline)) {
        const AtP at_p(p.P, p.ldp, (int64_t)rt * SIZE, p.rows, c, end);
        const AtQ at_q(p.Q, p.ldq, (int64_t)ot * SIZE, EPI == kEpiProb ? p.loss.outs : p.outs, c,
                       kTail ? min(end, p.q_end) : end);
        if constexpr (LOADS) {
            load_tile(at_p, p.ldp, lds[buf][0], wave, lane);
            load_tile(at_q, p.ldq, lds[buf][1], wave, lane);
        } else {
            fetch_tile<T>(at_p, p.ldp, held_p, wave, lane);
            fetch_tile<T>(at_q, p.ldq, held_q, wave, lane);
        }
    };
    auto put = [&](int buf) __attribute__((always_inline)) {
        if constexpr (!LOADS) {
            put_tile<PT, SIZE, S::waves>(held_p, lds[buf][0], wave, lane);
            put_tile<QT, SIZE, S::waves>(held_q, lds[buf][1], wave, lane);
        }
    };
    int buf = 0;
    int64_t tile = blockIdx.x;
    tile_of(p, tile, rt, ot);
    if (begin < end) {
        load(begin, 0);
        put(0);
    }
    // A workgroup's tiles one after another: the next one's first step is on its
    // way during the epilogue.
    for (; tile < total; tile += gridDim.x) {
        const int64_t row0 = (int64_t)rt * SIZE, out0 = (int64_t)ot * SIZE;
        const bool with_sums = kSums && ot == 0 && wo == 0;
        const int32_t this_rt = rt;
        // (kLoss) of row threadIdx.x: to LDS behind the loop's first barrier, which waits
        // for loads anyway (written here, they cost every tile a latency: 16,384 x 512 ->
        // 100,003 1.97 ms so, 2.16)
        RowInfo own{-1, 0.f, 0.f};
        if constexpr (kLoss) {
            const int64_t row = row0 + threadIdx.x;
            if (threadIdx.x < SIZE && row < p.rows) {
                const int64_t t = p.loss.target[row] - p.loss.first;
                own.t = t >= 0 && t < (EPI == kEpiProb ? p.loss.outs : p.outs) ? (int32_t)t : -1;
                if constexpr (EPI == kEpiProb) {
                    own.lse = p.loss.lse[row];
                    own.f = p.loss.f[row];
                }
            }
        }
        f4 acc[kNo][kNr], col[kSums ? kNr : 1];
#pragma unroll
        for (int j = 0; j < kNr; ++j) {
            if constexpr (kSums) col[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kNo; ++i) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        if constexpr (kLoss) {   // the bias is what the sums begin with (registers)
            if (p.bias) {
                const T* bias = reinterpret_cast<const T*>(p.bias);
                const int64_t outs = EPI == kEpiProb ? p.loss.outs : p.outs;
#pragma unroll
                for (int i = 0; i < kNo; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const int64_t at = out0 + S::outs * wo + 16 * i + 4 * g + v;
                        const float z = at < outs ? (float)bias[at] : 0.f;
#pragma unroll
                        for (int j = 0; j < kNr; ++j) acc[i][j][v] = z;
                    }
            }
        }
        for (int64_t c = begin; c < end; c += kStep, buf ^= 1) {
            // this tile has landed (loads into LDS are waited for by hand: the barrier
            // does not), and the last one's readers are done
            __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
            __syncthreads();
            if (kLoss && c == begin && threadIdx.x < SIZE) info[threadIdx.x] = own;
            if (c + kStep < end) load(c + kStep, buf ^ 1);
            const char* pt = lds[buf][0];
            const char* qt = lds[buf][1];
            v8 a[kStep / 32][kNo], b[kStep / 32][kNr];
            auto read = [&](int f) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < kNo; ++i) a[f][i] = fragment<T, QT, SIZE>(qt, kNo * wo + i, f, lane);
#pragma unroll
                for (int j = 0; j < kNr; ++j) b[f][j] = fragment<T, PT, SIZE>(pt, kNr * wr + j, f, lane);
            };
            // both halves' operands at once (128: 4 % faster) where there are registers;
            // 256: the second half's between the first half's products (4,096 x 4,096 of
            // 4,096 rows 111 us, 120 one after another; dW's take too many registers)
            constexpr bool kBoth = SIZE != 256 && LOADS, kBetween = SIZE == 256 && !PT;
            read(0);
            if constexpr (kBoth || kBetween) {
                __builtin_amdgcn_sched_barrier(0);
                read(1);
                if constexpr (kBoth) __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int f = 0; f < kStep / 32; ++f) {
                if (!kBoth && !kBetween && f) read(f);
                if constexpr (SIZE == 256 && PT) __builtin_amdgcn_s_setprio(1);   // (4 % faster so)
#pragma unroll
                for (int j = 0; j < kNr; ++j)
#pragma unroll
                    for (int i = 0; i < kNo; ++i)
                        acc[i][j] = Half<T>::mfma(a[f][i], b[f][j], acc[i][j]);
                if constexpr (kBetween) {
                    if (f == 0) {
#pragma unroll
                        for (int q = 0; q < kNo + kNr; ++q) {
                            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // an LDS read
                            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);   // two products
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if constexpr (kSums) {
                    if (with_sums) {
#pragma unroll
                        for (int j = 0; j < kNr; ++j) col[j] = Half<T>::mfma(ones, b[f][j], col[j]);
                    }
                }
                if constexpr (SIZE == 256 && PT) __builtin_amdgcn_s_setprio(0);
            }
            if (c + kStep < end) put(buf ^ 1);
        }
        constexpr int kLanes = S::outs / 8;      // lanes per row of the block, 8 outputs each
        constexpr int kRowsAtOnce = kWave / kLanes, kTurns = 16 / kRowsAtOnce;
        const int64_t out = out0 + S::outs * wo + 8 * (lane % kLanes);
        auto row_of = [&](int j, int v) __attribute__((always_inline)) -> int64_t {
            return row0 + S::rows * wr + 16 * j + v * kRowsAtOnce + lane / kLanes;
        };
        // The residual's (dy's) rows, 64 asked for ahead (a wait for each 16 rows:
        // 32,768 x 1,024 -> 4,096, gelu's slope 444 us, 379 so); not LOADS: where they
        // are used, the next step holds the registers.
        constexpr bool kEnds = EPI == kEpiForward || EPI == kEpiSlope;
        constexpr int kAhead = !(kEnds && LOADS) ? 1 : kNr < 4 ? kNr : 4;
        v8 bias = {}, res[kAhead][kTurns] = {};
        auto residual = [&](int j, int v) __attribute__((always_inline)) -> v8 {
            const int64_t row = row_of(j, v);
            if (!p.R || row >= p.rows) return v8{};
            return load8<T, FAST>(reinterpret_cast<const T*>(p.R) + row * p.ldr + out, p.outs - out);
        };
        if constexpr (kEnds) {
            if (p.bias)
                bias = load8<T, FAST>(reinterpret_cast<const T*>(p.bias) + out, p.outs - out);
            if constexpr (LOADS) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
#pragma unroll
                    for (int v = 0; v < kTurns; ++v) res[j][v] = residual(j, v);
            }
        }
        // the next tile's first step goes to `buf`, the epilogue's stages to the other
        __syncthreads();
        if (tile + gridDim.x < total) {
            tile_of(p, tile + gridDim.x, rt, ot);
            if (begin < end) load(begin, buf);
        }

        if constexpr (EPI == kEpiLse) {
            // a lane's outputs of a row: 16 i + 4 g + v of the wave's
            const int64_t left = p.outs - out0 - S::outs * wo;
            float2* blocks = p.loss.blocks + ((int64_t)(out0 / SIZE) * S::wave_outs + wo) * p.rows;
#pragma unroll
            for (int j = 0; j < kNr; ++j) {
                const int in = S::rows * wr + 16 * j + r;
                const int64_t row = row0 + in;
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int i = 0; i < kNo; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        if (left < S::outs && 16 * i + 4 * g + v >= left) acc[i][j][v] = -INFINITY;
                        top = __builtin_fmaxf(top, acc[i][j][v]);
                    }
                top = row_max4(top);
                const float mu = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int i = 0; i < kNo; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) sum += fast_exp2((acc[i][j][v] - mu) * kLog2eF);
                sum += __shfl_xor(sum, 16, kWave);
                sum += __shfl_xor(sum, 32, kWave);
                if (g == 0 && row < p.rows) blocks[row] = make_float2(top, sum);
                const int t = info[in].t - (int)(out0 + S::outs * wo);
                if (__ballot(info[in].t >= 0 && t >= 0 && t < S::outs && row < p.rows)) {
                    float z = 0.f;
#pragma unroll
                    for (int i = 0; i < kNo; ++i)
#pragma unroll
                        for (int v = 0; v < 4; ++v) z = t == 16 * i + 4 * g + v ? acc[i][j][v] : z;
                    if (info[in].t >= 0 && t >= 0 && t < S::outs && ((t >> 2) & 3) == g && row < p.rows)
                        p.loss.picked[row] = z;
                }
                __builtin_amdgcn_sched_barrier(0);   // (registers)
            }
            if (tile + gridDim.x < total && begin < end) put(buf);
            continue;
        }
        float* stage = reinterpret_cast<float*>(&lds[buf ^ 1][0][0]) + wave * 16 * kOutRow;
        float sum[8] = {};
        float* part = kPart ? reinterpret_cast<float*>(p.C) + (int64_t)blockIdx.y * p.rows * p.outs
                            : nullptr;
#pragma unroll
        for (int j = 0; j < kNr; ++j) {
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < kNo; ++i)
                *reinterpret_cast<f4*>(&stage[r * kOutRow + 16 * i + 4 * g]) = acc[i][j];
            wave_lds_order();
#pragma unroll
            for (int v = 0; v < kTurns; ++v) {
                const int rr = v * kRowsAtOnce + lane / kLanes;
                const float* src = &stage[rr * kOutRow + 8 * (lane % kLanes)];
                const f4 lo = *reinterpret_cast<const f4*>(src), hi = *reinterpret_cast<const f4*>(src + 4);
                const int64_t row = row_of(j, v);
                if constexpr (kPart) {
                    if (row < p.rows && out < p.outs) {
                        float* dst = part + row * p.outs + out;
                        if constexpr (EPI == kEpiAdd) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (out + k < p.outs) {
                                    const float x = k < 4 ? lo[k & 3] : hi[k & 3];
                                    dst[k] = p.add ? dst[k] + x : x;
                                }
                        } else if constexpr (FAST) {
                            *reinterpret_cast<f4*>(dst) = lo;
                            *reinterpret_cast<f4*>(dst + 4) = hi;
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (out + k < p.outs) dst[k] = k < 4 ? lo[k & 3] : hi[k & 3];
                        }
                    }
                } else if constexpr (EPI == kEpiProb) {
                    const RowInfo of = info[S::rows * wr + 16 * j + rr];
                    if (row < p.rows && out < p.outs) {
                        // (9 operations a value, one exponential among them, as many as the
                        // products of 64 steps take; 14 of them: 97 us for 16,384 x 512 ->
                        // 4,096, where nothing overlaps them)
                        float d[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                        each(d, [&](float z) { return fast_exp2((z - of.lse) * kLog2eF); });
                        const int t = of.t - (int)out;
                        if (t >= 0 && t < 8 && of.t >= 0) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) d[k] -= k == t ? 1.f : 0.f;
                        }
                        // (0 where f is, whatever z)
                        each(d, [&](float x) { return of.f == 0.f ? 0.f : x * of.f; });
                        if (out0 + SIZE > p.loss.outs) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) d[k] = out + k < p.loss.outs ? d[k] : 0.f;
                        }
                        if (p.sums) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) sum[k] += d[k];
                        }
                        typedef float f8 __attribute__((ext_vector_type(8)));
                        const v8 dz = __builtin_convertvector(
                            (f8{d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7]}), v8);
                        T* dst = reinterpret_cast<T*>(p.C) + row * p.outs + out;   // (whole pieces)
                        *reinterpret_cast<v8*>(dst) = dz;
                    }
                } else {
                    v8 other = {};
                    if constexpr (kEnds && LOADS) {
                        other = res[j % kAhead][v];
                        if (j + kAhead < kNr) res[j % kAhead][v] = residual(j + kAhead, v);
                    } else if constexpr (kEnds) {
                        other = residual(j, v);
                    }
                    finish8<T, EPI, FAST>(p, row, out, lo, hi, bias, other, sum);
                }
            }
        }
        if constexpr (EPI == kEpiSlope || EPI == kEpiProb) {
            if (p.sums) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
#pragma unroll
                    for (int off = kLanes; off < kWave; off <<= 1)
                        sum[k] += __shfl_xor(sum[k], off, kWave);
                    if (lane < kLanes && out + k < p.outs)
                        p.sums[((int64_t)this_rt * 2 + wr) * p.outs + out + k] = sum[k];
                }
            }
        }
        if constexpr (kSums) {
            if (with_sums && g == 0) {   // (every row of the ones' product is the sums)
#pragma unroll
                for (int j = 0; j < kNr; ++j) {
                    const int64_t row = row0 + S::rows * wr + 16 * j + r;
                    if (row < p.rows) p.sums[(int64_t)blockIdx.y * p.rows + row] = col[j][0];
                }
            }
        }
        if (tile + gridDim.x < total && begin < end) put(buf);
    }
}

// Splits of a product added: `count` values, and (db) the sums that came with them.
// WAYS 1: a thread for each value; 4: a wave for each quarter of the splits of 64
// values, the quarters added in order.  (50 splits of 128 x 512: 26 us and 10; one of
// 4,096 x 4,096: 35 and 90.  So 4 from 9 splits on, more than one turn of loads.)
__device__ __forceinline__ float split_sum(const float* __restrict__ at, int64_t stride,
                                           int32_t first, int32_t end)
{
    float s = 0.f;
    for (int32_t k = first; k < end; k += 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k + i < end ? at[(k + i) * stride] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x[i];
    }
    return s;
}
template <typename T, int WAYS>
__global__ void __launch_bounds__(256)
join_splits(const float* __restrict__ parts, int64_t count, int32_t splits, T* __restrict__ out,
            const float* __restrict__ sums, int64_t nsums, T* __restrict__ db)
{
    constexpr int kValues = 256 / WAYS;
    const int t = threadIdx.x % kValues, way = threadIdx.x / kValues;
    const int64_t i = (int64_t)blockIdx.x * kValues + t;
    const int32_t per = (splits + WAYS - 1) / WAYS, first = way * per, end = min(splits, first + per);
    float s = 0.f;
    if (i < count) s = split_sum(parts + i, count, first, end);
    else if (i < count + nsums) s = split_sum(sums + i - count, nsums, first, end);
    if constexpr (WAYS > 1) {
        __shared__ float lds[WAYS][kValues];
        lds[way][t] = s;
        __syncthreads();
        if (way) return;
#pragma unroll
        for (int w = 1; w < WAYS; ++w) s += lds[w][t];
    }
    if (i < count) out[i] = (T)s;
    else if (i < count + nsums) db[i - count] = (T)s;
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
        for (int64_t i = r0 + part; i < r1; i += 64) {
            float x[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = in[min(i + 4 * k, r1 - 1) * cols + col];
#pragma unroll
            for (int k = 0; k < 16; ++k) s += i + 4 * k < r1 ? x[k] : 0.f;
        }
    lds[part][threadIdx.x % 64] = s;
    __syncthreads();
    if (part == 0 && col < cols) {
        const int t = threadIdx.x;
        out[blockIdx.y * cols + col] = (OUT)((lds[0][t] + lds[1][t]) + (lds[2][t] + lds[3][t]));
    }
}

// ------------------------------------------------------------------ launches

// Where the tiles of 256 serve: elsewhere they would need more registers than
// there are.
constexpr bool has_256(int way, int epi)
{
    return way != kAny && epi != kEpiPartSums && epi != kEpiPlainSums;
}

// Size of the tiles and splits of the contraction, by what each choice would take:
// full waves of workgroups at the rate that a large product reaches (900, 760 and
// 580 TFLOP/s), 128 steps more for a tile's beginning and end, and for splits a
// launch and their sums' bytes at 8 TB/s (they stay in the Infinity Cache); twice the
// time where an operand's rows are no whole pieces.
// (Microseconds with 64, 128, 256, chosen; forward: 8,192 x 1,024 -> 1,024 32, 25,
// 40, 25; 200,003 x 512 -> 128 53, 55, 84, 53; 2,048 x 2,048 -> 2,048 28, 28, 49, 28;
// 1,024 x 1,024 -> 1,024 12, 16, 25, 12.  The rates are those at which these choices
// were measured; tiles of 256 have become faster since, so that their estimates are high:
// 344 us for 32,768 x 1,024 -> 4,096, which takes 268, and 157 for 4,096 cubed, 112.)
struct Tiling {
    int32_t tile, splits;
};
static inline Tiling tiling(int64_t rows, int64_t outs, int64_t depth, int64_t least, bool odd,
                     bool weights, bool sums = false)
{
    struct Kind {
        int32_t tile;
        int64_t slots;   // workgroups at once
        double alone;    // time of one of them alone on its CU, of that beside others
        double rate;     // multiplications per microsecond, full chip
    };
    const Kind kinds[] = {{256, 256, 1.0, 450e6}, {128, 512, 0.76, 380e6},
                          {64, 1280, 0.45, weights ? 230e6 : 290e6}};
    Tiling best{64, 1};
    double best_time = 1e300;
    for (const Kind& k : kinds) {
        if (k.tile == 256 && (odd || (weights && sums))) continue;
        const int64_t n = ceil_div(rows, k.tile) * ceil_div(outs, k.tile);
        for (int64_t s = 1; s <= 256 && (s == 1 || depth / s >= least); s += s < 4 ? 1 : s / 4) {
            // (a wave that is not full is shorter as far as workgroups share CUs)
            const double part = (double)(n * s % k.slots) / k.slots;
            const double waves = (double)(n * s / k.slots) + (part > 0 ? std::max(part, k.alone) : 0);
            double time = waves * k.slots * k.tile * k.tile * ((double)depth / s + 128) / k.rate;
            if (odd) time *= 2;   // (rows that are no whole pieces)
            if (s > 1) time += 3.0 + (double)rows * outs * (8 * s + 2) / 8e6;
            if (time < best_time) {
                best_time = time;
                best = Tiling{k.tile, (int32_t)s};
            }
        }
    }
    return best;
}
constexpr int64_t kForwardLeast = 512, kWeightLeast = 256;
constexpr int64_t kDbOuts = 8;   // columns of the product that db alone takes

static inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static inline int32_t tile_size(const Tiling& t, int way, int epi)
{
    return has_256(way, epi) ? t.tile : std::min(t.tile, 128);
}

// Workgroups of each split: as many as are resident at once, a multiple of eight (XCDs).
static inline int64_t workgroups_of(int64_t tiles, int32_t tile, int32_t splits)
{
    const int64_t resident = tile == 256 ? 256 : tile == 128 ? 512 : 1280;
    return std::min(tiles, std::max<int64_t>(8, resident / splits / 8 * 8));
}

template <typename T, bool PT, bool QT, int EPI, int WAY>
static void launch_tiles(GemmParams p, int32_t tile, hipStream_t st)
{
    p.row_tiles = (int32_t)ceil_div(p.rows, tile);
    p.out_tiles = (int32_t)ceil_div(p.outs, tile);
    p.split = ceil_div(ceil_div(p.depth, p.splits), 64) * 64;
    const dim3 grid((unsigned)workgroups_of((int64_t)p.row_tiles * p.out_tiles, tile, p.splits),
                    (unsigned)p.splits);
    if (tile == 64)
        hipLaunchKernelGGL((gemm_kernel<T, PT, QT, 64, EPI, WAY>), grid, dim3(256), 0, st, p);
    else if (tile == 128)
        hipLaunchKernelGGL((gemm_kernel<T, PT, QT, 128, EPI, WAY>), grid, dim3(256), 0, st, p);
    else if constexpr (has_256(WAY, EPI))
        hipLaunchKernelGGL((gemm_kernel<T, PT, QT, 256, EPI, WAY>), grid, dim3(512), 0, st, p);
}

// Offsets in a tile within 31 bits, and kWay's pieces.  (kTiles for forward products
// only, 2,000 x 2,000 -> 2,001 39 us so, 68 as kAny: in the others the outputs' number is
// that of an operand's columns.)
static inline Way way_of(const GemmParams& p, bool pt = false, bool qt = false)
{
    auto rows_ok = [](const char* x, int64_t ld) {
        return ((uintptr_t)x & 15) == 0 && ld % 8 == 0 && ld < (1 << 22);
    };
    const int64_t pcols = pt ? p.rows : p.depth, qcols = qt ? p.outs : p.depth;
    if (!rows_ok(p.P, p.ldp) || !rows_ok(p.Q, p.ldq) || pcols % 8 != 0 || qcols % 8 != 0) return kAny;
    if (p.outs % 8 == 0 && ((uintptr_t)p.C & 15) == 0 && (!p.bias || ((uintptr_t)p.bias & 15) == 0) &&
        (!p.R || rows_ok(p.R, p.ldr)))
        return kWhole;
    return pt || qt ? kAny : kTiles;
}

template <typename T, bool PT, bool QT, int EPI>
static inline f3s_status launch_gemm(GemmParams p, const Tiling& t, hipStream_t st)
{
    p.splits = t.splits;
    if (ceil_div(p.rows, t.tile) * ceil_div(p.outs, t.tile) >= ((int64_t)1 << 31)) {
        set_error("linear: too many tiles");
        return F3S_EUNSUPPORTED;
    }
    const Way way = way_of(p, PT, QT);
    const int32_t tile = tile_size(t, way, EPI);
    if (way == kWhole) launch_tiles<T, PT, QT, EPI, kWhole>(p, tile, st);
    else if (way == kAny) launch_tiles<T, PT, QT, EPI, kAny>(p, tile, st);
    else if constexpr (!PT && !QT) launch_tiles<T, PT, QT, EPI, kTiles>(p, tile, st);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

}  // namespace f3s
