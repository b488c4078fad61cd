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
    constexpr bool kPart = EPI == kEpiPart || EPI == kEpiPartSums;
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
        const AtQ at_q(p.Q, p.ldq, (int64_t)ot * SIZE, p.outs, c, end);
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
        f4 acc[kNo][kNr], col[kSums ? kNr : 1];
#pragma unroll
        for (int j = 0; j < kNr; ++j) {
            if constexpr (kSums) col[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kNo; ++i) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        for (int64_t c = begin; c < end; c += kStep, buf ^= 1) {
            // this tile has landed (loads into LDS are waited for by hand: the barrier
            // does not), and the last one's readers are done
            __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
            __syncthreads();
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
        if constexpr (EPI == kEpiSlope) {
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

constexpr int64_t kFewRows = 64, kManyRows = 48 * 1024;
constexpr int64_t kSumShares = 64, kSumRows = 512;

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
static Tiling tiling(int64_t rows, int64_t outs, int64_t depth, int64_t least, bool odd,
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

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static int32_t tile_size(const Tiling& t, int way, int epi)
{
    return has_256(way, epi) ? t.tile : std::min(t.tile, 128);
}

// Workgroups of each split: as many as are resident at once, a multiple of eight (XCDs).
static int64_t workgroups_of(int64_t tiles, int32_t tile, int32_t splits)
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
static Way way_of(const GemmParams& p, bool pt = false, bool qt = false)
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
static f3s_status launch_gemm(GemmParams p, const Tiling& t, hipStream_t st)
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
