// norm.hip -- layer norm and its gradient, rows of any width, binary16, bfloat16
// and float32 with float32 sums.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   dx = r (dh - mean dh - h mean (dh h)),  dh = dy w
//   dw = sum over the rows of dy h,  db = sum over the rows of dy
//
// What bounds it is one read of x (and dy) and one write of y (dx).  A row stays in
// the registers of the lanes that share it, 16-byte pieces of it each: 8 to 64 lanes
// of a wave, several rows side by side, or a whole workgroup.  So the variance is of
// the differences from the mean, with no second read.  The grid is what is resident
// at once: a workgroup goes from row to row, the next row's loads on their way, with
// w and b (and the sums of dw and db) in registers; its share of those sums goes to
// a line of its own, and a second launch adds the lines in order: no atomics, the
// same bits from run to run.
// A row that is no whole number of pieces ends in a piece that begins where the
// last V values do: it holds some values twice, which count once in the sums.
#include <algorithm>

#include "half_types.hpp"

namespace f3s {

struct NormParams {
    const char* x;
    const char* dy;
    const void* w;        // [C] or NULL (ones)
    const void* b;        // [C] or NULL (zeros)
    char* y;              // y; dx (NULL: not wanted)
    float* stats;         // [n][2]: m, r (forward: NULL: not kept)
    float* parts;         // [workgroups][2][C], backward (NULL: dw and db not wanted)
    int64_t ldx, lddy;    // values between rows
    int64_t n;
    int32_t C;
    int32_t wide_weights; // w and b are float32
    float eps;
};

template <typename T>
struct Pieces {
    static constexpr int V = 16 / sizeof(T);
    typedef T Raw __attribute__((ext_vector_type(16 / sizeof(T))));
};
template <typename R>
struct __attribute__((packed, aligned(2))) AnyPlace {
    R v;
};

// Where piece `num` of a row of C values begins, and how many of its values belong
// to the piece before (V: there is no such piece).  (C >= V)
template <int V>
struct Place {
    int32_t start, skip;
    __device__ __forceinline__ Place(int32_t num, int32_t C)
    {
        start = min(num * V, C - V);
        skip = min(num * V - start, V);
    }
};

// (SMALL: C may be below V)
template <typename T, bool SMALL>
__device__ __forceinline__ typename Pieces<T>::Raw load_piece(const T* row, int32_t start, int32_t C)
{
    typedef typename Pieces<T>::Raw Raw;
    if (!SMALL || C >= Pieces<T>::V) return reinterpret_cast<const AnyPlace<Raw>*>(row + start)->v;
    Raw r = {};
#pragma unroll
    for (int k = 0; k < Pieces<T>::V; ++k)   // (start = C - V < 0: the row's values are the last C)
        if (start + k >= 0) r[k] = row[start + k];
    return r;
}
template <typename T, bool SMALL>
__device__ __forceinline__ void store_piece(T* row, int32_t start, int32_t C,
                                            const float (&v)[Pieces<T>::V])
{
    typedef typename Pieces<T>::Raw Raw;
    Raw r;
#pragma unroll
    for (int k = 0; k < Pieces<T>::V; ++k) r[k] = (T)v[k];
    if (!SMALL || C >= Pieces<T>::V) {
        reinterpret_cast<AnyPlace<Raw>*>(row + start)->v = r;
        return;
    }
#pragma unroll
    for (int k = 0; k < Pieces<T>::V; ++k)
        if (start + k >= 0) row[start + k] = r[k];
}
// w's or b's values beside a piece.
template <typename T, bool SMALL>
__device__ __forceinline__ void load_weights(const void* w, int32_t wide, int32_t start, int32_t C,
                                             float other, float (&out)[Pieces<T>::V])
{
    constexpr int V = Pieces<T>::V;
    if (!w) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = other;
    } else if (SMALL && C < V) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int32_t c = max(start + k, 0);
            out[k] = wide ? static_cast<const float*>(w)[c] : (float)static_cast<const T*>(w)[c];
        }
    } else if (wide) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            const f4 a =
                reinterpret_cast<const AnyPlace<f4>*>(static_cast<const float*>(w) + start + 4 * q)->v;
#pragma unroll
            for (int k = 0; k < 4; ++k) out[4 * q + k] = a[k];
        }
    } else {
        const typename Pieces<T>::Raw a = load_piece<T, false>(static_cast<const T*>(w), start, C);
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = (float)a[k];
    }
}

// Sum over the LANES lanes that share a row; every one of them gets it.
template <int CTRL>
__device__ __forceinline__ float plus_lane(float x)
{
    return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL,
                                                                  0xf, 0xf, true));
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x)
{
    x = plus_lane<0xb1>(x);                            // lane ^ 1
    x = plus_lane<0x4e>(x);                            // lane ^ 2
    x = plus_lane<0x141>(x);                           // the other four of eight
    if constexpr (LANES >= 16) x = plus_lane<0x140>(x);   // the other eight of 16
    if constexpr (LANES >= 32) {
        auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if constexpr (LANES >= 64) {
        auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return x;
}
// N sums at once; a workgroup's through `lds`, which the sum before the last may
// still be read from, but no earlier one (a barrier lies between).
template <int LANES, int N>
__device__ __forceinline__ void row_sums_of(float (&x)[N], float (*lds)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lanes_sum<(LANES < 64 ? LANES : 64)>(x[i]);
    if constexpr (LANES > 64) {
        const int wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave][i] = x[i];
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
#pragma unroll
        for (int v = 0; v < LANES / kWave; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] += lds[v][i];
    }
}

// For the compiler new values: what was made of the old ones is not held.
template <typename R>
__device__ __forceinline__ void anew_piece(R& a, R& b)
{
    u4 x = __builtin_bit_cast(u4, a), y = __builtin_bit_cast(u4, b);
    asm volatile("" : "+v"(x), "+v"(y));
    a = __builtin_bit_cast(R, x);
    b = __builtin_bit_cast(R, y);
}

constexpr int norm_threads(int lanes) { return lanes > 256 ? lanes : 256; }

template <typename T, int LANES, int NP>
__global__ void __launch_bounds__(norm_threads(LANES)) norm_fwd_kernel(const NormParams p)
{
    constexpr int V = Pieces<T>::V, kRows = norm_threads(LANES) / LANES;
    typedef typename Pieces<T>::Raw Raw;
    __shared__ float lds[2][16][1];
    const int l = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int32_t C = p.C;
    const T* x = reinterpret_cast<const T*>(p.x);
    int32_t start[NP], skip[NP];
    float w[NP][V], b[NP][V];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const Place<V> at(l + j * LANES, C);
        start[j] = at.start;
        skip[j] = at.skip;
        load_weights<T, LANES == 8>(p.w, p.wide_weights, at.start, C, 1.f, w[j]);
        load_weights<T, LANES == 8>(p.b, p.wide_weights, at.start, C, 0.f, b[j]);
    }
    const float inv = 1.f / (float)C;
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + sub;
    Raw next[NP];
    auto load = [&](int64_t r) __attribute__((always_inline)) {
        const T* src = x + min(r, p.n - 1) * p.ldx;
#pragma unroll
        for (int j = 0; j < NP; ++j) next[j] = load_piece<T, LANES == 8>(src, start[j], C);
    };
    load(row);
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.n; base += step, row += step) {
        float v[NP][V], s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[j][k] = (float)next[j][k];
                s[0] += k >= skip[j] ? v[j][k] : 0.f;
            }
        if (base + step < p.n) load(row + step);
        row_sums_of<LANES, 1>(s, lds[0]);
        const float m = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[j][k] -= m;
                s[0] = k >= skip[j] ? __builtin_fmaf(v[j][k], v[j][k], s[0]) : s[0];
            }
        row_sums_of<LANES, 1>(s, lds[1]);
        const float r = 1.f / __builtin_sqrtf(__builtin_fmaf(s[0], inv, p.eps));
        if (row < p.n) {
            T* dst = reinterpret_cast<T*>(p.y) + row * C;
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                if (skip[j] >= V) continue;
#pragma unroll
                for (int k = 0; k < V; ++k) v[j][k] = __builtin_fmaf(v[j][k] * r, w[j][k], b[j][k]);
                store_piece<T, LANES == 8>(dst, start[j], C, v[j]);
            }
            if (p.stats && l == 0) *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(m, r);
        }
    }
}

template <typename T, int LANES, int NP>
__global__ void __launch_bounds__(norm_threads(LANES)) norm_bwd_kernel(const NormParams p)
{
    constexpr int V = Pieces<T>::V, kThreads = norm_threads(LANES), kRows = kThreads / LANES;
    typedef typename Pieces<T>::Raw Raw;
    __shared__ float lds[2][16][2];
    const int l = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int32_t C = p.C;
    const T* x = reinterpret_cast<const T*>(p.x);
    const T* dy = reinterpret_cast<const T*>(p.dy);
    int32_t start[NP], skip[NP];
    float w[NP][V], dw[NP][V], db[NP][V];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const Place<V> at(l + j * LANES, C);
        start[j] = at.start;
        skip[j] = at.skip;
        load_weights<T, LANES == 8>(p.w, p.wide_weights, at.start, C, 1.f, w[j]);
#pragma unroll
        for (int k = 0; k < V; ++k) dw[j][k] = db[j][k] = 0.f;
    }
    const float inv = 1.f / (float)C;
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + sub;
    Raw nx[NP], ny[NP];
    float2 stat;
    auto load = [&](int64_t r) __attribute__((always_inline)) {
        r = min(r, p.n - 1);
        const T* sx = x + r * p.ldx;
        const T* sy = dy + r * p.lddy;
        stat = *reinterpret_cast<const float2*>(p.stats + 2 * r);
#pragma unroll
        for (int j = 0; j < NP; ++j) nx[j] = load_piece<T, LANES == 8>(sx, start[j], C);
#pragma unroll
        for (int j = 0; j < NP; ++j) ny[j] = load_piece<T, LANES == 8>(sy, start[j], C);
    };
    // (the next row's loads ahead where the registers are there for them)
    constexpr bool kAhead = LANES < 1024 || NP < 4;
    if (kAhead) load(row);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < p.n; base += step, row += step, turn ^= 1) {
        if (!kAhead) load(row);
        const float m = stat.x, r = stat.y;
        const bool there = row < p.n;
        Raw cx[NP], cy[NP];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            cx[j] = nx[j];
            cy[j] = ny[j];
        }
        if (kAhead && base + step < p.n) load(row + step);
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float g = there ? (float)cy[j][k] : 0.f, h = ((float)cx[j][k] - m) * r;
                if (there) {   // (0 x inf of a row that is another's again)
                    dw[j][k] = __builtin_fmaf(g, h, dw[j][k]);
                    db[j][k] += g;
                }
                if (k >= skip[j]) {
                    s[0] = __builtin_fmaf(g, w[j][k], s[0]);
                    s[1] = __builtin_fmaf(g * w[j][k], h, s[1]);
                }
            }
        if (p.y) {
            row_sums_of<LANES, 2>(s, lds[turn]);
            const float s0 = s[0] * inv, s1 = s[1] * inv;
            if (there) {
                T* dst = reinterpret_cast<T*>(p.y) + row * C;
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if (skip[j] >= V) continue;
                    // (h and dh again, from the pieces: held, they are 32 registers of a
                    // workgroup's 128 where rows are widest)
                    if constexpr (LANES >= 1024) anew_piece(cx[j], cy[j]);
                    float dx[V];
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        dx[k] = r * ((float)cy[j][k] * w[j][k] - s0 - ((float)cx[j][k] - m) * r * s1);
                    store_piece<T, LANES == 8>(dst, start[j], C, dx);
                }
            }
        }
    }
    if (!p.parts) return;
    float* out = p.parts + (int64_t)blockIdx.x * 2 * C;
    if constexpr (LANES >= 256) {
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (skip[j] < V && start[j] + k >= 0) {   // (a value held twice: the same sum twice)
                    out[start[j] + k] = dw[j][k];
                    out[C + start[j] + k] = db[j][k];
                }
    } else {
        // the wave's rows side by side, then the four waves in order
        constexpr int kCols = LANES * NP * V;
        __shared__ float sums[kThreads / kWave][kCols];
        const int wave = threadIdx.x / kWave;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (which) __syncthreads();
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float s = which ? db[j][k] : dw[j][k];
#pragma unroll
                    for (int off = LANES; off < kWave; off <<= 1) s += __shfl_xor(s, off, kWave);
                    if (threadIdx.x % kWave < LANES && skip[j] < V && start[j] + k >= 0)
                        sums[wave][start[j] + k] = s;
                }
            __syncthreads();
            for (int32_t c = threadIdx.x; c < C; c += kThreads)
                out[which * C + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
        }
    }
}

// Rows too wide for a workgroup's registers: read again for each sum (from the
// caches, as a rule).
constexpr int kWideThreads = 1024;
__device__ __forceinline__ float block_sum(float x, float* lds)
{
    x = lanes_sum<64>(x);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
    __syncthreads();
    float s = 0.f;
    for (int v = 0; v < kWideThreads / kWave; ++v) s += lds[v];
    return s;
}
// f(start, skip) for the thread's pieces of a row.  (C >= V here)
template <int V, typename F>
__device__ __forceinline__ void own_pieces(int32_t C, F f)
{
    for (int32_t num = threadIdx.x; (int64_t)num * V < C; num += kWideThreads) {
        const Place<V> at(num, C);
        f(at.start, at.skip);
    }
}
template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_fwd(const NormParams p)
{
    constexpr int V = Pieces<T>::V;
    typedef typename Pieces<T>::Raw Raw;
    __shared__ float lds[kWideThreads / kWave];
    const int32_t C = p.C;
    const float inv = 1.f / (float)C;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
        T* y = reinterpret_cast<T*>(p.y) + row * C;
        float s = 0.f;
        own_pieces<V>(C, [&](int32_t start, int32_t skip) {
            const Raw a = load_piece<T, false>(x, start, C);
#pragma unroll
            for (int k = 0; k < V; ++k) s += k >= skip ? (float)a[k] : 0.f;
        });
        const float m = block_sum(s, lds) * inv;
        s = 0.f;
        own_pieces<V>(C, [&](int32_t start, int32_t skip) {
            const Raw a = load_piece<T, false>(x, start, C);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = (float)a[k] - m;
                s = k >= skip ? __builtin_fmaf(d, d, s) : s;
            }
        });
        const float r = 1.f / __builtin_sqrtf(__builtin_fmaf(block_sum(s, lds), inv, p.eps));
        own_pieces<V>(C, [&](int32_t start, int32_t) {
            const Raw a = load_piece<T, false>(x, start, C);
            float w[V], b[V], v[V];
            load_weights<T, false>(p.w, p.wide_weights, start, C, 1.f, w);
            load_weights<T, false>(p.b, p.wide_weights, start, C, 0.f, b);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = __builtin_fmaf(((float)a[k] - m) * r, w[k], b[k]);
            store_piece<T, false>(y, start, C, v);
        });
        if (p.stats && threadIdx.x == 0)
            *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(m, r);
    }
}
template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_dx(const NormParams p)
{
    constexpr int V = Pieces<T>::V;
    typedef typename Pieces<T>::Raw Raw;
    __shared__ float lds[kWideThreads / kWave];
    const int32_t C = p.C;
    const float inv = 1.f / (float)C;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
        const T* dy = reinterpret_cast<const T*>(p.dy) + row * p.lddy;
        T* dx = reinterpret_cast<T*>(p.y) + row * C;
        const float m = p.stats[2 * row], r = p.stats[2 * row + 1];
        float s0 = 0.f, s1 = 0.f;
        own_pieces<V>(C, [&](int32_t start, int32_t skip) {
            const Raw a = load_piece<T, false>(x, start, C), d = load_piece<T, false>(dy, start, C);
            float w[V];
            load_weights<T, false>(p.w, p.wide_weights, start, C, 1.f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float dh = k >= skip ? (float)d[k] * w[k] : 0.f;
                s0 += dh;
                s1 = k >= skip ? __builtin_fmaf(dh, ((float)a[k] - m) * r, s1) : s1;
            }
        });
        s0 = block_sum(s0, lds) * inv;
        s1 = block_sum(s1, lds) * inv;
        own_pieces<V>(C, [&](int32_t start, int32_t) {
            const Raw a = load_piece<T, false>(x, start, C), d = load_piece<T, false>(dy, start, C);
            float w[V], v[V];
            load_weights<T, false>(p.w, p.wide_weights, start, C, 1.f, w);
#pragma unroll
            for (int k = 0; k < V; ++k)
                v[k] = r * ((float)d[k] * w[k] - s0 - ((float)a[k] - m) * r * s1);
            store_piece<T, false>(dx, start, C, v);
        });
    }
}
// 256 columns of blockIdx.y's share of the rows.
template <typename T>
__global__ void __launch_bounds__(256) norm_wide_sums(const NormParams p)
{
    const int32_t C = p.C, c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    const int64_t per = (p.n + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = blockIdx.y * per, r1 = min(p.n, r0 + per);
    float dw = 0.f, db = 0.f;
    for (int64_t row = r0; row < r1; ++row) {
        const float g = (float)reinterpret_cast<const T*>(p.dy)[row * p.lddy + c];
        const float v = (float)reinterpret_cast<const T*>(p.x)[row * p.ldx + c];
        dw = __builtin_fmaf(g, (v - p.stats[2 * row]) * p.stats[2 * row + 1], dw);
        db += g;
    }
    float* out = p.parts + (int64_t)blockIdx.y * 2 * C;
    out[c] = dw;
    out[C + c] = db;
}

// dw and db from the workgroups' lines, in 64 bits: 16 columns by 64 parts of the
// lines, the parts added in order.  (1,024 lines of 512: 20 us by 16 parts, whose loads
// were waited for four times, 7 so.)
constexpr int kJoinParts = 64;
template <typename W>
__global__ void __launch_bounds__(16 * kJoinParts)
norm_join(const float* __restrict__ parts, int32_t lines, int32_t C, W* __restrict__ dw,
          W* __restrict__ db)
{
    __shared__ double lds[kJoinParts][17];
    const int col = threadIdx.x % 16, part = threadIdx.x / 16;
    const int64_t c = (int64_t)blockIdx.x * 16 + col, width = 2 * (int64_t)C;
    const int32_t per = (lines + kJoinParts - 1) / kJoinParts, first = part * per,
                  end = min(lines, first + per);
    double s = 0.0;
    if (c < width) {
        for (int32_t i = first; i < end; i += 16) {
            float x[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = i + k < end ? parts[(i + k) * width + c] : 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += x[k];
        }
    }
    lds[part][col] = s;
    __syncthreads();
    if (part == 0 && c < width) {
        double t = 0.0;
#pragma unroll
        for (int v = 0; v < kJoinParts; ++v) t += lds[v][col];
        W* out = c < C ? dw : db;
        if (out) out[c < C ? c : c - C] = (W)(float)t;
    }
}

__global__ void warm_norm_kernel() {}

hipError_t warm_norm(hipStream_t s)
{
    hipLaunchKernelGGL(warm_norm_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

// ------------------------------------------------------------------ launches

constexpr int64_t kCus = 256;

// Lanes and pieces of a row; lanes 0: too wide.
struct NormShape {
    int32_t lanes, pieces;
};
static NormShape norm_shape(int64_t C, int32_t dtype, bool backward)
{
    const int64_t have = ceil_div(C, dtype == F3S_F32 ? 4 : 8);
    for (int32_t lanes : {8, 16, 32, 64})
        if (have <= lanes) return {lanes, 1};
    if (have <= 128) return {64, 2};
    // (the gradient's registers: 32 values a lane in 512 lanes; 16 in 1,024 spilled, 12,736
    // wide in bfloat16 486 us a step, 298 so)
    if (backward && dtype != F3S_F32 && have > 1024 && have <= 2048) return {512, 4};
    for (int32_t lanes : {256, 512, 1024})
        for (int32_t pieces : {1, 2})
            if ((pieces == 2 || lanes == 256) && have <= (int64_t)lanes * pieces)
                return {lanes, pieces};
    // (float32: four pieces are as many values as 16-bit types' two; of the gradient's
    // registers 11 spill)
    if (dtype == F3S_F32 && have <= 4096) return {1024, 4};
    return {0, 0};
}

// Workgroups: what is resident at once, eight waves per SIMD forward; backward no
// more than four, whose lines are read again.
static int64_t norm_groups(const NormShape& s, int64_t n, bool backward)
{
    const int64_t threads = s.lanes ? norm_threads(s.lanes) : kWideThreads;
    const int64_t rows = s.lanes ? threads / s.lanes : 1;
    return std::min(ceil_div(n, rows), kCus * (backward ? 1024 : 2048) / threads);
}
static int64_t wide_lines(int64_t n) { return std::min<int64_t>(n, 64); }

static size_t norm_bytes(int64_t n, int64_t C, int32_t dtype)
{
    const NormShape s = norm_shape(C, dtype, true);
    return sizeof(float) * 2 * (size_t)C * (size_t)(s.lanes ? norm_groups(s, n, true) : wide_lines(n));
}

template <typename T, bool BACKWARD, typename F>
static void with_shape(const NormShape& s, F go)
{
    auto one = [&](auto lanes, auto pieces) {
        if (s.lanes == decltype(lanes)::value && s.pieces == decltype(pieces)::value) go(lanes, pieces);
    };
    std::integral_constant<int, 1> p1;
    std::integral_constant<int, 2> p2;
    one(std::integral_constant<int, 8>{}, p1);
    one(std::integral_constant<int, 16>{}, p1);
    one(std::integral_constant<int, 32>{}, p1);
    one(std::integral_constant<int, 64>{}, p1);
    one(std::integral_constant<int, 64>{}, p2);
    one(std::integral_constant<int, 256>{}, p1);
    one(std::integral_constant<int, 256>{}, p2);
    one(std::integral_constant<int, 512>{}, p2);
    std::integral_constant<int, 4> p4;
    if constexpr (BACKWARD && sizeof(T) == 2) one(std::integral_constant<int, 512>{}, p4);
    else one(std::integral_constant<int, 1024>{}, p2);
    if constexpr (sizeof(T) == 4) one(std::integral_constant<int, 1024>{}, p4);
}

template <typename T>
static void norm_forward(const NormParams& p, int32_t dtype, hipStream_t st)
{
    const NormShape s = norm_shape(p.C, dtype, false);
    const dim3 grid((unsigned)norm_groups(s, p.n, false));
    if (!s.lanes) {
        hipLaunchKernelGGL((norm_wide_fwd<T>), grid, dim3(kWideThreads), 0, st, p);
        return;
    }
    with_shape<T, false>(s, [&](auto lanes, auto pieces) {
        constexpr int L = decltype(lanes)::value, N = decltype(pieces)::value;
        hipLaunchKernelGGL((norm_fwd_kernel<T, L, N>), grid, dim3(norm_threads(L)), 0, st, p);
    });
}

template <typename T>
static void norm_backward(const NormParams& p, int32_t dtype, void* dw, void* db, hipStream_t st)
{
    const NormShape s = norm_shape(p.C, dtype, true);
    const dim3 grid((unsigned)norm_groups(s, p.n, true));
    int64_t lines = grid.x;
    if (!s.lanes) {
        if (p.y) hipLaunchKernelGGL((norm_wide_dx<T>), grid, dim3(kWideThreads), 0, st, p);
        lines = wide_lines(p.n);
        if (p.parts)
            hipLaunchKernelGGL((norm_wide_sums<T>),
                               dim3((unsigned)ceil_div(p.C, 256), (unsigned)lines), dim3(256), 0, st,
                               p);
    } else {
        with_shape<T, true>(s, [&](auto lanes, auto pieces) {
            constexpr int L = decltype(lanes)::value, N = decltype(pieces)::value;
            hipLaunchKernelGGL((norm_bwd_kernel<T, L, N>), grid, dim3(norm_threads(L)), 0, st, p);
        });
    }
    if (!p.parts) return;
    const dim3 join((unsigned)ceil_div(2 * (int64_t)p.C, 16));
    if (p.wide_weights)
        hipLaunchKernelGGL((norm_join<float>), join, dim3(16 * kJoinParts), 0, st, p.parts,
                           (int32_t)lines, p.C, static_cast<float*>(dw), static_cast<float*>(db));
    else
        hipLaunchKernelGGL((norm_join<T>), join, dim3(16 * kJoinParts), 0, st, p.parts,
                           (int32_t)lines, p.C, static_cast<T*>(dw), static_cast<T*>(db));
}

template <typename W>
__global__ void __launch_bounds__(256) norm_zero(W* __restrict__ a, W* __restrict__ b, int32_t C)
{
    const int32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c < C && a) a[c] = (W)0.f;
    if (c < C && b) b[c] = (W)0.f;
}

static f3s_status check_norm(int64_t n, int64_t C, int32_t dtype, int32_t weight_dtype,
                             const char* who)
{
    if (n < 0 || C < 1 || dtype < F3S_F16 || dtype > F3S_F32 ||
        (weight_dtype != dtype && weight_dtype != F3S_F32)) {
        set_error(std::string(who) + ": bad size or type (weights are of x's type or float32)");
        return F3S_EINVAL;
    }
    if (C >= ((int64_t)1 << 24) || n >= ((int64_t)1 << 40)) {
        set_error(std::string(who) + ": width below 2^24, n below 2^40");
        return F3S_EUNSUPPORTED;
    }
    return F3S_OK;
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_layer_norm_workspace(int64_t n, int64_t C, int32_t dtype, int64_t* bytes)
{
    F3S_REQUIRE(bytes, "f3s_layer_norm_workspace: NULL pointer");
    F3S_TRY(check_norm(n, C, dtype, dtype, "f3s_layer_norm_workspace"));
    *bytes = n == 0 ? 0 : (int64_t)norm_bytes(n, C, dtype);
    return F3S_OK;
}

f3s_status f3s_layer_norm_fwd(const void* X, int64_t x_stride, const void* W, const void* B, void* Y,
                              float* stats, int64_t n, int64_t C, float eps, int32_t dtype,
                              int32_t weight_dtype, void* stream)
{
    F3S_TRY(check_norm(n, C, dtype, weight_dtype, "f3s_layer_norm_fwd"));
    if (n == 0) return F3S_OK;
    F3S_REQUIRE(X && Y && x_stride >= C && ((uintptr_t)stats & 7) == 0,
                "f3s_layer_norm_fwd: NULL or misaligned pointer, or a row stride below the width");
    F3S_TRY(require_device());
    clear_error();
    NormParams p{};
    p.x = static_cast<const char*>(X);
    p.ldx = x_stride;
    p.w = W;
    p.b = B;
    p.y = static_cast<char*>(Y);
    p.stats = stats;
    p.n = n;
    p.C = (int32_t)C;
    p.eps = eps;
    p.wide_weights = weight_dtype == F3S_F32;
    hipStream_t st = as_stream(stream);
    if (dtype == F3S_F16) norm_forward<_Float16>(p, dtype, st);
    else if (dtype == F3S_BF16) norm_forward<__bf16>(p, dtype, st);
    else norm_forward<float>(p, dtype, st);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

f3s_status f3s_layer_norm_bwd(const void* X, int64_t x_stride, const void* W, const float* stats,
                              const void* dY, int64_t dy_stride, void* dX, void* dW, void* dB,
                              int64_t n, int64_t C, int32_t dtype, int32_t weight_dtype,
                              void* workspace, int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_norm(n, C, dtype, weight_dtype, "f3s_layer_norm_bwd"));
    F3S_REQUIRE(n == 0 || (X && dY && stats && x_stride >= C && dy_stride >= C &&
                           ((uintptr_t)stats & 7) == 0),
                "f3s_layer_norm_bwd: NULL or misaligned pointer, or a row stride below the width");
    const bool sums = dW || dB;
    F3S_REQUIRE(n == 0 || !sums ||
                    (workspace && ((uintptr_t)workspace & 15) == 0 &&
                     workspace_bytes >= (int64_t)norm_bytes(n, C, dtype)),
                "f3s_layer_norm_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    if (n == 0) {
        const dim3 grid((unsigned)ceil_div(C, 256));
        if (sums && weight_dtype == F3S_F32)
            hipLaunchKernelGGL((norm_zero<float>), grid, dim3(256), 0, st, static_cast<float*>(dW),
                               static_cast<float*>(dB), (int32_t)C);
        else if (sums)   // (both 16-bit types' zero)
            hipLaunchKernelGGL((norm_zero<_Float16>), grid, dim3(256), 0, st,
                               static_cast<_Float16*>(dW), static_cast<_Float16*>(dB), (int32_t)C);
        F3S_HIP(hipGetLastError());
        return F3S_OK;
    }
    if (!sums && !dX) return F3S_OK;
    NormParams p{};
    p.x = static_cast<const char*>(X);
    p.ldx = x_stride;
    p.dy = static_cast<const char*>(dY);
    p.lddy = dy_stride;
    p.w = W;
    p.y = static_cast<char*>(dX);
    p.stats = const_cast<float*>(stats);
    p.parts = sums ? static_cast<float*>(workspace) : nullptr;
    p.n = n;
    p.C = (int32_t)C;
    p.wide_weights = weight_dtype == F3S_F32;
    if (dtype == F3S_F16) norm_backward<_Float16>(p, dtype, dW, dB, st);
    else if (dtype == F3S_BF16) norm_backward<__bf16>(p, dtype, dW, dB, st);
    else norm_backward<float>(p, dtype, dW, dB, st);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

}  // extern "C"
