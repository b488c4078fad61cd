// edge_attention.hip -- softmax attention over a graph's edges with capped scores and
// a bias by distance, and its gradient, on the compiled column lists of a plan
// (attention.hip).
//
// Per head 64 dims; over the edges i -> j
//   x = scale q(i).k(j),  s = cap tanh(x / cap) - slope |pos(i) - pos(j)|
//   p = softmax of s,  o(i) = sum_j p v(j)            (rows without edges: 0)
// and, for a gradient do(i), with g = do(i).v(j), D(i) = sum_j p g and
// c = 1 - tanh^2(x / cap),
//   dq(i) = scale sum_j p (g - D) c k(j),  dk(j) = scale sum_i p (g - D) c q(i)
//   dv(j) = sum_i p do(i),  dslope = -sum p (g - D) |pos(i) - pos(j)|
//
// Three passes of one shape: a wave takes a window of 16 rows of one head and streams
// the rows at the other ends of its edges past it, 32 a chunk, two 128-byte rows each:
//   forward  k, v past q:       m, l and the sums of p v
//   rows     k, v past q, do:   the sums of p g' c k, p c k, p g' and p, g' = g - the mean
//            of the row's first g: dq = scale (sum p g' c k - D' sum p c k) needs no second
//            sweep for D, and nothing of o is kept from the forward pass but a log-sum-exp
//   columns  q, do past k, v, on the plan of the reversed edges: dk, dv; no atomics
// What bounds them is the random 256 bytes per edge and head.
//
// Weights go to the matrix cores as the sum of two 16-bit values (split8): rounded
// once, every weight of a row would be off by up to half a step of the type before
// the result is rounded itself.  In binary16 what can be far below 1 is scaled, as
// kLift and range_update say.  Sums and softmax statistics are in float32.
//
// A value that is infinite or NaN reaches, through the matrix cores, rows of its
// window that have no edge to it (0 x inf).  So a window whose sums are not finite is
// done again, edge by edge without them (slow_row): in the same launch where teams
// share windows, else in the one that joins segments, which finds none as a rule.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstddef>

#include "edge_stream.hpp"

namespace f3s {

constexpr int kHeadHalves = kD;                    // of a row in LDS
constexpr int kEdgeHeadBytes = kRowBytes;          // q, k, v, o of one head
constexpr float kLog2e = 1.4426950408889634f;

enum EdgePass : int { kForward = 0, kRows = 1, kColumns = 2 };

struct EdgeParams {
    EdgeRows x1, x2;        // streamed: k and v; q and do on the reversed edges
    EdgeRows own1, own2;    // the window's own rows: q and do; k and v
    EdgeRows out1, out2;    // o; dq; dk and dv
    const float* slopes;    // [H] (dims > 0)
    const float* positions; // [n][dims]
    float* lse;             // [n][H], log2; forward: written (NULL: not)
    float* stats;           // [n][H][stat_words]: lse, D and the position
    float* slope_parts;     // [H][slope_windows]
    float* dslopes;         // [H]
    int32_t slope_windows;  // of the rows' pass
    const Item* items;
    const int32_t* chunk_base;
    const uint32_t* columns;
    const SplitInfo* splits;
    float* partials;
    uint32_t* odd;          // [items][H]: sums that are not finite
    int32_t* slot_item;     // [slots]
    int64_t num_items, num_split;
    int32_t W, n, H, dims, stat_words;
    int32_t xcd_contiguous, team;
    // the lists' references: node indices, or node * H * 128 (below kNoRow);
    // node = ((ref >> shift) * magic) >> 31, magic 2^31 or ceil(2^31 / H), which is
    // exact below 2^25
    uint32_t ref_shift, ref_magic, no_ref;
    float scale, scale_log2;
    float cap;              // 0: none
    float cap_in, cap_log2; // scale / cap; cap log2(e)
};

// What a node and head have beside their rows, for the columns' pass: one line for lse,
// D and the position (2, 4 or 8 words), where a position of its own would be another.
static inline int32_t stat_words(int32_t dims) { return dims == 0 ? 2 : dims <= 2 ? 4 : 8; }

// The forward pass's weights are 2^kLazy at most: in binary16 raised to 2^14, so that the
// small ones of a row of many edges keep their bits.  (3,000 equal weights of 2^-18 beside
// one of 1, unraised: their sum was off by 2^-9 of itself.)
template <typename T>
constexpr float kSoftLog2 = Half<T>::kRange ? 14.f - kLazy : 0.f;

// A wave's sums, tiles of 16 dims, lane (g, r) holding dims 16 t + 4 g + v of row r in
// tile t (v: the element), and its share of row r's sums of weights.
//   forward: tiles 0-3 sum p v, scaled by 2^-x, x the running maximum (binary16: by
//            kSoftLog2 more); y: l, as they
//   rows:    0-3 sum p g' c k, scaled by 2^-x; 4-7 sum p c k; y: sum p g', z: sum p,
//            yd, zd: the same times the distance; ref: g - g', mass: recentre()
//   columns: 0-3 sum ds q, scaled by 2^-x; 4-7 dv
template <int PASS>
struct EdgeState {
    static constexpr int tiles = PASS == kForward ? 4 : 8;
    f4 acc[tiles];
    float x, y, z, yd, zd, ref, mass;
};
// floats of a published state
template <int PASS>
constexpr int state_floats() { return (EdgeState<PASS>::tiles + 2) * kWave * 4; }

template <int PASS>
__device__ __forceinline__ void clear(EdgeState<PASS>& s)
{
#pragma unroll
    for (int t = 0; t < s.tiles; ++t) s.acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    s.x = -INFINITY;
    s.y = s.z = s.yd = s.zd = 0.f;
    s.ref = s.mass = 0.f;
}

template <int PASS>
__device__ __forceinline__ void rescale(EdgeState<PASS>& s, float factor)
{
#pragma unroll
    for (int t = 0; t < 4; ++t) s.acc[t] *= factor;
}

// (rows) The least scale of sums that what moves a reference by x is added to: there it is
// 2^24, or less where 2 to the scale has no inverse.
__device__ __forceinline__ float scale_of(float x)
{
    return __builtin_fmaxf((float)(__builtin_amdgcn_frexp_expf(x) - 24), -100.f);
}

template <int PASS>
__device__ __forceinline__ void publish(const EdgeState<PASS>& s, float* dst, int lane)
{
#pragma unroll
    for (int t = 0; t < s.tiles; ++t) *reinterpret_cast<f4*>(&dst[(t * kWave + lane) * 4]) = s.acc[t];
    *reinterpret_cast<f4*>(&dst[(s.tiles * kWave + lane) * 4]) = f4{s.x, s.y, s.z, s.yd};
    dst[(s.tiles + 1) * kWave * 4 + lane] = s.zd;
    if constexpr (PASS == kRows) {
        dst[((s.tiles + 1) * 4 + 1) * kWave + lane] = s.ref;
        dst[((s.tiles + 1) * 4 + 2) * kWave + lane] = s.mass;
    }
}

// Takes a published state into s.
template <int PASS>
__device__ __forceinline__ void absorb(EdgeState<PASS>& s, const float* src, int lane)
{
    const f4 w = *reinterpret_cast<const f4*>(&src[(s.tiles * kWave + lane) * 4]);
    const float zd = src[(s.tiles + 1) * kWave * 4 + lane];
    f4 a[EdgeState<PASS>::tiles];   // (all on their way before the first is waited for)
#pragma unroll
    for (int t = 0; t < s.tiles; ++t)
        a[t] = *reinterpret_cast<const f4*>(&src[(t * kWave + lane) * 4]);
    const float ref = PASS == kRows ? src[((s.tiles + 1) * 4 + 1) * kWave + lane] : 0.f;
    const float mass = PASS == kRows ? src[((s.tiles + 1) * 4 + 2) * kWave + lane] : 0.f;
    __builtin_amdgcn_sched_barrier(0);
    float top = __builtin_fmaxf(s.x, w[0]);
    // (rows) the lighter one's sums move to the heavier one's reference
    const bool moves = mass > s.mass;   // (s does)
    const float apart = moves ? s.ref - ref : ref - s.ref;
    if (PASS == kRows && apart != 0.f) top = __builtin_fmaxf(top, scale_of(apart));
    const float mine = top == -INFINITY ? 0.f : fast_exp2(s.x - top);
    const float theirs = top == -INFINITY ? 0.f : fast_exp2(w[0] - top);
    rescale(s, mine);
    if constexpr (PASS == kForward) {
        s.y = s.y * mine + w[1] * theirs;
    } else {
        if constexpr (PASS == kRows) {
            s.y = __builtin_fmaf(apart, moves ? s.z : w[2], s.y);
            s.yd = __builtin_fmaf(apart, moves ? s.zd : zd, s.yd);
            const float by = apart != 0.f ? apart * fast_exp2(-top) : 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t) s.acc[t] += by * (moves ? s.acc[4 + t] : a[4 + t]);
            s.ref = moves ? ref : s.ref;
            s.mass = __builtin_fmaxf(mass, s.mass);
        }
        s.y += w[1];
        s.z += w[2];
        s.yd += w[3];
        s.zd += zd;
    }
    s.x = top;
#pragma unroll
    for (int t = 0; t < s.tiles; ++t) s.acc[t] += t < 4 ? a[t] * theirs : a[t];
}

// A wave's memory: a chunk's rows of x1 and x2, 128 bytes each, a row's 16-byte pieces
// in an order of its own (piece p at p ^ edge_swizzle(row)): 16 rows' pieces of one
// number, which the products with the window's rows read, and four rows' pairs of
// pieces, which the transposing reads take, then lie in distinct banks without padding.
// One record of the lists (offsets into x1 and x2, or node indices; row masks) per
// chunk, two in turn, and what the chunk's slots have beside their rows.
// 9,728 bytes: 16 waves fit a CU's 160 KB.
__device__ __forceinline__ int edge_swizzle(int row) { return (row & 6) | ((row >> 3) & 1); }
struct EdgeRecord {
    uint32_t at1[kChunk], at2[kChunk], rm[kChunk];
};
struct __align__(128) EdgeLds {
    _Float16 x1[kChunk * kHeadHalves];
    _Float16 x2[kChunk * kHeadHalves];
    EdgeRecord rec[2];
    float pos[kChunk * 4];    // dims 1: the first 32; else x, y, z, - of each slot
    float stats[kChunk * 2];
};
static_assert(sizeof(EdgeLds) <= 10240, "16 waves per CU");
static_assert(4 * sizeof(EdgeLds) >= 2 * sizeof(float) * state_floats<kRows>(),
              "a team's memory holds two states");
constexpr uint32_t kEdgeStage = sizeof(_Float16) * kChunk * kHeadHalves;   // x2 after x1
constexpr uint32_t kEdgeHalf = kEdgeStage / 2;                             // 16 rows

// Where a lane reads and writes in a stage (addresses in LDS).
struct EdgePlaces {
    uint32_t row;     // piece g of row r
    uint32_t column;  // what lane r of group g hands the transposing read of tile 0
    uint32_t write;   // piece lane % 8 of row lane / 8
};
// (the addresses of all pieces come from these by exclusive or with constants, made
// where they are used: held in registers, they would be some thirty)
__device__ __forceinline__ void held(EdgePlaces& p)
{
    asm volatile("" : "+v"(p.row), "+v"(p.column), "+v"(p.write));
}
__device__ __forceinline__ EdgePlaces edge_places(const _Float16* stage, int lane)
{
    const int g = lane >> 4, r = lane & 15, i = r >> 2, c = r & 3;
    const uint32_t base = (uint32_t)(uintptr_t)(LdsPtr)stage;
    return EdgePlaces{base + 128 * r + 16 * (g ^ edge_swizzle(r)),
                      base + 128 * (4 * g + i) + 16 * ((c >> 1) ^ edge_swizzle(4 * g + i)) + 8 * (c & 1),
                      base + 128 * (lane >> 3) + 16 * ((lane & 7) ^ edge_swizzle(lane >> 3))};
}

// Rows 8 i + lane / 8, i = 0 .. 3, from the lane's pieces.  (Rows 8 apart differ in the
// last bit of their order.)
template <typename V>
__device__ __forceinline__ void edge_write(const EdgePlaces& p, uint32_t stage, const V (&x)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) lds_write(((p.write ^ (16 * (i & 1))) + stage) + 1024 * i, x[i]);
}

// 16 rows of a stage times the window's rows.
template <typename T>
__device__ __forceinline__ f4 edge_products(const EdgePlaces& p, uint32_t stage,
                                            const typename Half<T>::v8 (&own)[2])
{
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < 2; ++f)
        s = Half<T>::mfma(lds_read<typename Half<T>::v8>((p.row ^ (64 * f)) + stage), own[f], s);
    return s;
}

// acc[t] += sum over the chunk's slots of hi + lo (the lane's slots of row r) times
// dims 16 t .. of the stage's rows.  Each group of 16 lanes hands four rows of 16
// values to the transposing read, lane r its piece of row r / 4, and receives column
// r of them; twice, for slots 4 g .. and 16 + 4 g ...
template <typename T>
__device__ __forceinline__ void edge_mix(const EdgePlaces& p, uint32_t stage,
                                         const float (&w)[8], f4* acc)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* lds4;
    typename Half<T>::v8 hi, lo, x[4];
    split8<T>(w, hi, lo);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t at = (p.column ^ (32 * t)) + stage;
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)at);
        const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at + kEdgeHalf));
        x[t] = __builtin_bit_cast(typename Half<T>::v8,
                                  s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = Half<T>::mfma(x[t], hi, acc[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = Half<T>::mfma(x[t], lo, acc[t]);
}

// tanh, to 3e-7 of itself: by its series up to 0.3 (the next term is 6e-8 of it
// there), else from one exponential, whose 1e-7 are 4e-7 of 0.29.
constexpr float kNear = 0.3f;
__device__ __forceinline__ float tanh_near(float x)
{
    const float t = x * x;
    float s = __builtin_fmaf(t, 62.f / 2835.f, -17.f / 315.f);
    s = __builtin_fmaf(s, t, 2.f / 15.f);
    s = __builtin_fmaf(s, t, -1.f / 3.f);
    return __builtin_fmaf(x * t, s, x);
}
__device__ __forceinline__ float tanh_far(float x)
{
    return __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + fast_exp2(2.f * kLog2e * x)), 1.f);
}

// Scores in log2 units from the products of their rows, and c = 1 - tanh^2.  (Scores
// are small beside their cap as a rule: the exponential only where one of the wave's
// is not.)
template <int N>
__device__ __forceinline__ void edge_scores(const EdgeParams& p, float (&s)[N], float (&c)[N])
{
    if (p.cap == 0.f) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            c[j] = 1.f;
            s[j] *= p.scale_log2;
        }
        return;
    }
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        s[j] *= p.cap_in;
        most = __builtin_fmaxf(most, __builtin_fabsf(s[j]));
    }
    if (__ballot(!(most < kNear))) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            s[j] = __builtin_fabsf(s[j]) < kNear ? tanh_near(s[j]) : tanh_far(s[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = tanh_near(s[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        c[j] = __builtin_fmaf(-s[j], s[j], 1.f);
        s[j] *= p.cap_log2;
    }
}

struct Position {
    float x, y, z;
};
// The square of a distance, and the distance by a power of two of its largest
// coordinate, so that no square leaves the type.
__device__ __forceinline__ float squared(const Position& a, float x, float y, float z)
{
    const float dx = a.x - x, dy = a.y - y, dz = a.z - z;
    return __builtin_fmaf(dz, dz, __builtin_fmaf(dy, dy, dx * dx));
}
__device__ __forceinline__ float distance(const Position& a, float x, float y, float z)
{
    float dx = a.x - x, dy = a.y - y, dz = a.z - z;
    const int e = __builtin_amdgcn_frexp_expf(
        __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(dx), __builtin_fabsf(dy)), __builtin_fabsf(dz)));
    dx = __builtin_amdgcn_ldexpf(dx, -e);
    dy = __builtin_amdgcn_ldexpf(dy, -e);
    dz = __builtin_amdgcn_ldexpf(dz, -e);
    return __builtin_amdgcn_ldexpf(
        __builtin_amdgcn_sqrtf(__builtin_fmaf(dz, dz, __builtin_fmaf(dy, dy, dx * dx))), e);
}
// Infinite coordinates: of a window's rows as +inf, at the edges' other ends as -inf, so
// that the distance of two nodes of which either is infinitely far is infinite, not NaN.
__device__ __forceinline__ Position facing(Position a, float infinity)
{
    a.x = __builtin_fabsf(a.x) == INFINITY ? infinity : a.x;
    a.y = __builtin_fabsf(a.y) == INFINITY ? infinity : a.y;
    a.z = __builtin_fabsf(a.z) == INFINITY ? infinity : a.z;
    return a;
}
__device__ __forceinline__ Position position_of(const EdgeParams& p, int64_t node)
{
    Position a{0.f, 0.f, 0.f};
    if (p.dims) {
        const float* at = p.positions + node * p.dims;
        a.x = at[0];
        if (p.dims > 1) a.y = at[1];
        if (p.dims > 2) a.z = at[2];
    }
    return a;
}
// The distances of row r's node to the lane's slots 16 t + 4 g ..
__device__ __forceinline__ void distances(const EdgeLds& L, const Position& own, int dims, int t,
                                          int lane, float (&d)[4])
{
    const int slot = 16 * t + 4 * (anew(lane) >> 4);
    if (dims == 1) {
        const f4 a = *reinterpret_cast<const f4*>(&L.pos[slot]);
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = __builtin_fabsf(own.x - a[j]);
        return;
    }
    float least = INFINITY, most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f4 a = *reinterpret_cast<const f4*>(&L.pos[4 * (slot + j)]);
        d[j] = squared(own, a[0], a[1], a[2]);
        least = __builtin_fminf(least, d[j]);
        most = __builtin_fmaxf(most, d[j]);
    }
    if (__ballot(least < 0x1p-100f || !(most < 0x1p126f))) {   // (a loop's 0 among them)
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            const f4 a = *reinterpret_cast<const f4*>(&L.pos[4 * (slot + j)]);
            const float x = distance(own, a[0], a[1], a[2]);
            d[0] = j == 0 ? x : d[0];
            d[1] = j == 1 ? x : d[1];
            d[2] = j == 2 ? x : d[2];
            d[3] = j == 3 ? x : d[3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = __builtin_amdgcn_sqrtf(d[j]);
    }
}

// Scales weights of unknown size into binary16: a power of two per row, st.x, moved
// (and the sums that it scales with it) when a weight would come within a factor of
// four of the type's end, to put that weight at 2^3 to 2^4.
template <typename T, int PASS>
__device__ __forceinline__ void range_update(EdgeState<PASS>& st, float (&w)[8])
{
    if constexpr (Half<T>::kRange) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(w[j]));
        most = row_max4(most);
        // (2^x may be far below 2^-126: compare exponents)
        const float e = most > 0.f ? (float)__builtin_amdgcn_frexp_expf(most) : -INFINITY;
        if (__ballot(e > st.x + 14.f)) {
            if (e > st.x + 14.f) {
                const float x = __builtin_fminf(e, 128.f) - 4.f;
                rescale(st, fast_exp2(st.x - x));
                st.x = x;
            }
        }
        const int f = st.x == -INFINITY ? 0 : (int)-st.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_ldexpf(w[j], f);
    }
}

// Sum over the four lanes that hold a row.
__device__ __forceinline__ float row_sum4(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What the rows' pass takes from g: the mean of those so far, so that weights are rounded
// after what is common to them has been taken out.  (Values of mean 64 left an error of
// 1.6e-3 in bfloat16's dq, beside its own rounding's 1.65e-3, where sums of p g c k were
// rounded first.)  u, w: a chunk's p g' c and p c, in the sums' y and z already.  The mean
// is taken anew, and all sums moved to it, where the weights so far have become four times
// those of the last one: a far-off g of a small weight then does not stay what all others
// are taken from.
template <typename T, int PASS>
__device__ __forceinline__ void recentre(EdgeState<PASS>& st, float (&u)[8], const float (&w)[8])
{
    const float mass = row_sum4(st.z);
    if (!__ballot(mass > 4.f * st.mass)) return;
    const float away = row_sum4(st.y) / mass;
    if (!(mass > 4.f * st.mass && __builtin_fabsf(away) <= FLT_MAX)) return;
    if (st.mass > 0.f && away != 0.f) {
        float by = away;
        if constexpr (Half<T>::kRange) {
            const float x = __builtin_fmaxf(st.x, scale_of(away));
            rescale(st, fast_exp2(st.x - x));
            st.x = x;
            by *= fast_exp2(-x);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) st.acc[t] -= by * st.acc[4 + t];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = __builtin_fmaf(-away, w[j], u[j]);
    st.y = __builtin_fmaf(-away, st.z, st.y);
    st.yd = __builtin_fmaf(-away, st.zd, st.yd);
    st.ref += away;
    st.mass = mass;
}

// Rows of 64 values leave whole, through a stage of 16 rows: val(t) is the lane's part
// of tile t, dims 16 t + 4 g .. + 3.
template <typename T, typename F>
__device__ __forceinline__ void edge_store(const EdgeRows& out, _Float16* stage, int32_t w, int32_t n,
                                           uint32_t head_off, int lane, F val)
{
    typedef typename Half<T>::v8 v8;
    typedef typename Half<T>::v4 v4;
    const int g = lane >> 4, r = lane & 15;
    wave_lds_order();
#pragma unroll
    for (int t = 0; t < 4; ++t)
        *reinterpret_cast<v4*>(&stage[r * kHeadHalves + 8 * ((2 * t + (g >> 1)) ^ edge_swizzle(r)) +
                                      4 * (g & 1)]) = __builtin_convertvector(val(t), v4);
    wave_lds_order();
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int rr = 8 * v + (lane >> 3), piece = lane & 7;
        const v8 x = *reinterpret_cast<const v8*>(
            &stage[rr * kHeadHalves + 8 * (piece ^ edge_swizzle(rr))]);
        const int32_t row = w * 16 + rr;
        if (row < n)
            *reinterpret_cast<v8*>(const_cast<char*>(out.ptr) + row * out.stride + head_off +
                                   16 * piece) = x;
    }
    wave_lds_order();
}

// Whether a sum is not finite.
template <int PASS>
__device__ __forceinline__ bool odd_state(const EdgeState<PASS>& st)
{
    float odd = 0.f;   // (x - x is 0 for finite x, NaN otherwise)
#pragma unroll
    for (int t = 0; t < st.tiles; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) odd += st.acc[t][v] - st.acc[t][v];
    return __ballot(odd != 0.f) != 0;
}

// A window's results from its sums.
template <typename T, int PASS>
__device__ __forceinline__ void edge_finish(const EdgeParams& p, EdgeState<PASS>& st, _Float16* stage,
                                            int32_t w, int h, int lane)
{
    lane = anew(lane);
    const int g = lane >> 4, r = lane & 15;
    const int32_t row = w * 16 + r;
    const uint32_t head_off = (uint32_t)h * kEdgeHeadBytes;
    if constexpr (PASS == kForward) {
        const float l = over_groups(st.y);
        const float f = l != 0.f ? 1.f / l : 0.f;   // (a row of NaN is some)
        edge_store<T>(p.out1, stage, w, p.n, head_off, lane, [&](int t) {
            return l != 0.f ? st.acc[t] * f : f4{0.f, 0.f, 0.f, 0.f};
        });
        if (p.lse && g == 0 && row < p.n)
            p.lse[(int64_t)row * p.H + h] = l != 0.f ? st.x + (__log2f(l) - kSoftLog2<T>) : 0.f;
    } else if constexpr (PASS == kRows) {
        // The weights' own sum (1, but for the rounding of the log-sum-exp) divides.
        const float l = over_groups(st.z);
        const float i = l != 0.f ? 1.f / l : 0.f;
        const float d = over_groups(st.y) * i;   // (from the reference)
        const float f = fast_exp2(st.x);   // (0: unset)
        const float c = p.scale * i;
        edge_store<T>(p.out1, stage, w, p.n, head_off, lane,
                      [&](int t) { return c * (st.acc[t] * f - d * st.acc[4 + t]); });
        if (g == 0 && row < p.n)
            p.stats[((int64_t)row * p.H + h) * p.stat_words + 1] = l != 0.f ? d + st.ref : 0.f;
        if (p.dims) {
            // the window's share of dslope: rows 0 to 15 in one fixed order
            float s = row < p.n ? (over_groups(st.yd) - d * over_groups(st.zd)) * i : 0.f;
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor(s, off, kWave);
            if (lane == 0) p.slope_parts[(int64_t)h * p.slope_windows + w] = s;
        }
    } else {
        const float f = p.scale * fast_exp2(st.x);
        edge_store<T>(p.out1, stage, w, p.n, head_off, lane,
                      [&](int t) { return st.acc[t] * f; });
        edge_store<T>(p.out2, stage, w, p.n, head_off, lane,
                      [&](int t) { return st.acc[4 + t] * (1.f / kLift<T>); });
    }
}

// One row of a window edge by edge, lane d holding dim d, sums in float32 without
// products of zero: its results, and (rows) its share of dslope.  list(k) is the k-th
// of the window's items.
template <typename T, int PASS, typename F>
__device__ float slow_row(const EdgeParams& p, int32_t w, int h, int r, int nitems, F list, int lane)
{
    const int32_t row = w * 16 + r;
    if (row >= p.n) return 0.f;
    const int rbit = (r & 1) ? 16 + (r >> 1) : (r >> 1);
    const int64_t at = (int64_t)row * p.H + h;
    auto value = [&](const EdgeRows& x, int64_t node) -> float {
        return (float)reinterpret_cast<const T*>(x.ptr + node * x.stride)[h * kD + lane];
    };
    const float a = value(p.own1, row), b = PASS == kForward ? 0.f : value(p.own2, row);
    const Position own = facing(position_of(p, row), INFINITY);
    const float slope = p.dims ? p.slopes[h] * kLog2e : 0.f;
    const float lse = PASS == kRows ? p.lse[at] : 0.f;
    float m = -INFINITY, l = 0.f, pg = 0.f, pd = 0.f, pgd = 0.f;   // (uniform)
    float acc1 = 0.f, acc2 = 0.f;
    for (int k = 0; k < nitems; ++k) {
        const int32_t item = list(k);
        for (int32_t c = p.chunk_base[item]; c < p.chunk_base[item + 1]; ++c) {
            const uint32_t word = p.columns[(int64_t)c * 64 + lane];
            uint32_t slots = (uint32_t)(__ballot((word >> rbit) & 1u) >> 32);
            for (; slots; slots &= slots - 1) {
                const uint32_t ref =
                    (uint32_t)__builtin_amdgcn_readlane((int)word, __builtin_ctz(slots));
                const int64_t node =
                    (int64_t)(((uint64_t)(ref >> p.ref_shift) * p.ref_magic) >> 31);
                const float y1 = value(p.x1, node), y2 = value(p.x2, node);
                float dist = 0.f, score[1] = {wave_sum(a * y1)}, slopes_c[1];
                edge_scores(p, score, slopes_c);
                float s = score[0];
                const float slope_c = slopes_c[0];
                if (p.dims) {
                    const Position there = facing(position_of(p, node), -INFINITY);
                    dist = p.dims == 1 ? __builtin_fabsf(own.x - there.x)
                                       : distance(own, there.x, there.y, there.z);
                    s -= slope * dist;
                }
                if constexpr (PASS == kForward) {
                    const float top = s == s ? __builtin_fmaxf(m, s) : s;
                    if (top == -INFINITY) continue;
                    const float mine = fast_exp2(m - top), e = fast_exp2(s - top);
                    l = l * mine + e;
                    acc1 = acc1 * mine + e * y2;
                    m = top;
                } else if constexpr (PASS == kRows) {
                    const float e = fast_exp2(s - lse), g = wave_sum(b * y2);
                    if (e == 0.f) dist = 0.f;   // (an infinite one)
                    l += e;
                    pg += e * g;
                    pd += e * dist;
                    pgd += e * g * dist;
                    acc1 += e * g * slope_c * y1;
                    acc2 += e * slope_c * y1;
                } else {
                    const float2 st =
                        *reinterpret_cast<const float2*>(p.stats + (node * p.H + h) * p.stat_words);
                    const float e = fast_exp2(s - st.x), g = wave_sum(b * y2);
                    acc1 += e * (g - st.y) * slope_c * y1;
                    acc2 += e * y2;
                }
            }
        }
    }
    auto store = [&](const EdgeRows& out, float v) {
        reinterpret_cast<T*>(const_cast<char*>(out.ptr) + row * out.stride)[h * kD + lane] = (T)v;
    };
    if constexpr (PASS == kForward) {
        store(p.out1, l != 0.f ? acc1 / l : 0.f);
        if (p.lse && lane == 0) p.lse[at] = l != 0.f ? m + __log2f(l) : 0.f;
        return 0.f;
    } else if constexpr (PASS == kRows) {
        const float i = l != 0.f ? 1.f / l : 0.f, d = pg * i;
        store(p.out1, p.scale * i * (acc1 - d * acc2));
        if (lane == 0) p.stats[at * p.stat_words + 1] = d;
        return (pgd - d * pd) * i;
    } else {
        store(p.out1, p.scale * acc1);
        store(p.out2, acc2);
        return 0.f;
    }
}

constexpr int kEdgeWaves = 4;   // per workgroup
static_assert(kEdgeWaves == kTeamSmall, "a team fills its workgroup");

// A window by slow_row, its rows dealt to the workgroup's waves.  (Every thread of the
// workgroup calls it.)
template <typename T, int PASS, typename F>
__device__ void slow_window(const EdgeParams& p, int32_t w, int h, int nitems, F list, float* lds)
{
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    __syncthreads();
    for (int r = wave; r < 16; r += kEdgeWaves) {
        const float s = slow_row<T, PASS>(p, w, h, r, nitems, list, lane);
        if (PASS == kRows && lane == 0) lds[r] = s;
    }
    if constexpr (PASS == kRows) {
        __syncthreads();
        if (threadIdx.x == 0 && p.dims) {
            float s = 0.f;
            for (int r = 0; r < 16; ++r) s += lds[r];
            p.slope_parts[(int64_t)h * p.slope_windows + w] = s;
        }
        __syncthreads();
    }
}

// -sum of a head's windows' shares, by THREADS threads.
template <int THREADS>
__device__ __forceinline__ void sum_slopes(const float* __restrict__ src, int32_t W,
                                           float* __restrict__ out)
{
    __shared__ double lds[THREADS / kWave];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < W; i += 32 * THREADS) {
        float x[32];   // (in one batch: the loads' latency is all there is)
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = src[min(i + k * THREADS, (int64_t)W - 1)];
#pragma unroll
        for (int k = 0; k < 32; ++k) s += i + k * THREADS < W ? x[k] : 0.f;
    }
    s = wave_sum(s);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < THREADS / kWave; ++i) t += lds[i];
        *out = (float)-t;
    }
}

// TEAM: a window's four items are its workgroup's waves (small graphs); else a wave
// takes an item, a window or a segment of one.
template <typename T, int PASS, bool WIDE, bool TEAM>
__global__ void __launch_bounds__(kWave * kEdgeWaves) __attribute__((amdgpu_waves_per_eu(PASS == kForward ? 4 : 3)))
edge_kernel(const EdgeParams p)
{
    typedef typename Half<T>::v8 v8;
    __shared__ EdgeLds lds_all[kEdgeWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    EdgeLds& L = lds_all[wave];
    const uint32_t H = (uint32_t)p.H;
    const int32_t n = p.n;

    // ---- which item and head.  A scheduled plan's items are eight interleaved shares,
    // share x for XCD x, and the dispatcher deals workgroups to the XCDs in turn:
    // workgroup b takes items of share b % 8.  A natural-order plan's shares are
    // contiguous instead.
    uint32_t item, h;
    if constexpr (TEAM) {
        const uint32_t gb = (uint32_t)logical_block(p.xcd_contiguous);
        item = gb / H * kEdgeWaves + wave;
        h = gb % H;
    } else {
        const uint32_t xcd = blockIdx.x % kXcds, share = (uint32_t)((p.num_items + kXcds - 1) / kXcds);
        const uint32_t at = blockIdx.x / kXcds * kEdgeWaves + wave, i = at / H;
        h = at % H;
        item = p.xcd_contiguous ? xcd * share + i : i * kXcds + xcd;
        if (i >= share || item >= (uint32_t)p.num_items) return;
    }
    const u4 it = scalar_load(reinterpret_cast<const u4*>(p.items + item));
    const int32_t w = (int32_t)it[0], slot = (int32_t)it[3];
    if (w < 0 || w >= p.W) {   // (a team's four items alike)
        if (!TEAM && lane == 0) p.odd[item * H + h] = 0u;
        return;
    }
    const int32_t cb = scalar_load(p.chunk_base + item), ce = scalar_load(p.chunk_base + item + 1);

    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(p.x1.ptr, p.x1.bytes);
    const __amdgpu_buffer_rsrc_t r2 = make_rsrc(p.x2.ptr, p.x2.bytes);

    // ---- the window's own rows, in operand order: dims 32 f + 8 g .. of row r (rows
    // past the last are not stored) ----
    v8 o1[2], o2[2];
    const int32_t row = min(w * 16 + r, n - 1);
    {
        const char* src = p.own1.ptr + row * p.own1.stride + h * kEdgeHeadBytes + 16 * g;
#pragma unroll
        for (int f = 0; f < 2; ++f) o1[f] = *reinterpret_cast<const v8*>(src + 64 * f);
    }
    if constexpr (PASS != kForward) {
        const char* src = p.own2.ptr + row * p.own2.stride + h * kEdgeHeadBytes + 16 * g;
#pragma unroll
        for (int f = 0; f < 2; ++f) o2[f] = *reinterpret_cast<const v8*>(src + 64 * f);
    }
    const Position own = facing(position_of(p, row), INFINITY);
    const float slope = p.dims ? scalar_load(p.slopes + h) * kLog2e : 0.f;
    float lse = 0.f;
    if constexpr (PASS == kRows) {
        lse = p.lse[(int64_t)row * H + h];
        if (g == 0 && w * 16 + r < n && (!TEAM || wave == 0)) {
            float* to = p.stats + ((int64_t)row * H + h) * p.stat_words;
            to[0] = lse;
            if (p.dims) *reinterpret_cast<f2*>(to + 2) = f2{own.x, own.y};
            if (p.dims > 2) to[4] = own.z;
        }
        lse -= kLiftLog2<T>;
    }

    EdgePlaces at = edge_places(L.x1, lane);
    const uint32_t masks0 = (uint32_t)(uintptr_t)(LdsPtr)&L.rec[0].rm[0];
    v8 a[4], b[4];
    Position there{0.f, 0.f, 0.f};   // of slot lane % 32
    f2 stat = {0.f, 0.f};
    uint32_t word = 0;
    // A record's words, one per lane: 32 references, 32 masks.  (The lists end in spare
    // records.)
    auto fetch = [&](int32_t c) __attribute__((always_inline)) {
        return (p.columns + (int64_t)c * 64)[anew(lane)];
    };
    // Into the record of chunk c, and the loads of its slots.
    auto load = [&](int32_t c) __attribute__((always_inline)) {
        const int lane = anew(threadIdx.x % kWave);
        EdgeRecord& rec = L.rec[(c - cb) & 1];
        const uint32_t ref = __shfl(word, lane & 31, kWave);
        const bool none = ref >= p.no_ref;
        const uint32_t node = (uint32_t)(((uint64_t)(ref >> p.ref_shift) * p.ref_magic) >> 31);
        if (lane >= 32) {
            rec.rm[lane - 32] = word;
        } else if constexpr (WIDE) {
            rec.at1[lane] = none ? kNoIdx : node;
        } else {
            rec.at1[lane] = none ? kNoRow : node * (uint32_t)p.x1.stride;
            rec.at2[lane] = none ? kNoRow : node * (uint32_t)p.x2.stride;
        }
        wave_lds_order();
        const uint32_t extra = h * kEdgeHeadBytes + 16 * (lane & 7);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t at1 = rec.at1[8 * i + (lane >> 3)];
            if constexpr (WIDE) {
                a[i] = b[i] = v8{};
                if (at1 != kNoIdx) {
                    a[i] = *reinterpret_cast<const v8*>(p.x1.ptr + at1 * p.x1.stride + extra);
                    b[i] = *reinterpret_cast<const v8*>(p.x2.ptr + at1 * p.x2.stride + extra);
                }
            } else {
                a[i] = __builtin_bit_cast(
                    v8, __builtin_amdgcn_raw_buffer_load_b128(r1, at1 + extra, 0, 0));
            }
        }
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t at2 = rec.at2[8 * i + (lane >> 3)];
                b[i] = __builtin_bit_cast(
                    v8, __builtin_amdgcn_raw_buffer_load_b128(r2, at2 + extra, 0, 0));
            }
        }
        const int64_t i = none ? 0 : node;
        if constexpr (PASS == kColumns) {
            const float* from = p.stats + (i * H + h) * p.stat_words;
            if (p.dims) {
                const f4 x = *reinterpret_cast<const f4*>(from);
                stat = f2{x[0], x[1]};
                there.x = x[2];
                there.y = x[3];
                if (p.dims > 2) there.z = from[4];
            } else {
                stat = *reinterpret_cast<const f2*>(from);
            }
        } else if (p.dims) {
            there = position_of(p, i);
        }
    };

    EdgeState<PASS> st;
    clear(st);
    if (PASS != kForward && !Half<T>::kRange) st.x = 0.f;
    if (cb < ce) {
        word = fetch(cb);
        load(cb);
        word = fetch(cb + 1);
    }
    for (int32_t c = cb; c < ce; ++c) {
        const uint32_t masks = masks0 + ((c - cb) & 1) * (uint32_t)sizeof(EdgeRecord);
        held(at);
        edge_write(at, 0, a);
        edge_write(at, kEdgeStage, b);
        const int own_slot = anew(lane) & 31;
        if (p.dims) {
            const Position to = facing(there, -INFINITY);
            if (p.dims == 1) L.pos[own_slot] = to.x;
            else *reinterpret_cast<f4*>(&L.pos[4 * own_slot]) = f4{to.x, to.y, to.z, 0.f};
        }
        if constexpr (PASS == kColumns) *reinterpret_cast<f2*>(&L.stats[2 * own_slot]) = stat;
        wave_lds_order();
        if (c + 1 < ce) {
            load(c + 1);
            word = fetch(c + 2);   // (past the item's last: another's, or a spare one)
        }
        // Half of the slots at a time (registers): scores of slots 16 t + 4 g .. of row r,
        // and what the products after them take: w beside acc[4 ..] (forward: acc), u
        // beside acc[0 .. 3].
        float w8[8], u8[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            const f4 dots = edge_products<T>(at, kEdgeHalf * t, o1);
            float s[4] = {dots[0], dots[1], dots[2], dots[3]}, cc[4], dist[4];
            f4 gs;   // do . v
            if constexpr (PASS != kForward) gs = edge_products<T>(at, kEdgeStage + kEdgeHalf * t, o2);
            edge_scores(p, s, cc);
            if (p.dims) {
                distances(L, own, p.dims, t, lane, dist);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = __builtin_fmaf(-slope, dist[j], s[j]);
            }
            uint32_t on[4];
            attends_half(masks, t, lane, on);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float& w = w8[4 * t + j];
                [[maybe_unused]] float& u = u8[4 * t + j];
                if constexpr (PASS == kForward) {
                    w = where(on[j], s[j], -INFINITY);
                } else if constexpr (PASS == kRows) {
                    const float e = where(on[j], fast_exp2(lifted<T>(s[j] - lse, kLiftLog2<T> + 1.f)));
                    const float eg = where(on[j], e * (gs[j] - st.ref));
                    st.z += e;
                    st.y += eg;
                    if (p.dims) {
                        const float d = e != 0.f ? dist[j] : 0.f;   // (an infinite one's e is 0)
                        st.zd = __builtin_fmaf(e, d, st.zd);
                        st.yd = __builtin_fmaf(eg, d, st.yd);
                    }
                    w = where(on[j], e * cc[j]);
                    u = where(on[j], eg * cc[j]);
                } else {
                    const f2 of = *reinterpret_cast<const f2*>(&L.stats[2 * (16 * t + 4 * (anew(lane) >> 4) + j)]);
                    const float e = where(on[j], fast_exp2(lifted<T>(s[j] - of[0], 0.f)));
                    u = where(on[j], e * (gs[j] - of[1]) * cc[j]);
                    w = e * kLift<T>;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (PASS == kForward) {
            // the running maximum is moved when a chunk's exceeds it by more than kLazy
            float top = w8[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top = __builtin_fmaxf(top, w8[j]);
            top = row_max4(top);
            if (__ballot(top > st.x + kLazy)) {
                if (top > st.x + kLazy) {
                    const float corr = fast_exp2(st.x - top);
                    st.y *= corr;
                    rescale(st, corr);
                    st.x = top;
                }
            }
            const float mu = (st.x == -INFINITY ? 0.f : st.x) - kSoftLog2<T>;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w8[j] = fast_exp2(w8[j] - mu);
                st.y += w8[j];
            }
            edge_mix<T>(at, kEdgeStage, w8, st.acc);
        } else {
            if constexpr (PASS == kRows) recentre<T>(st, u8, w8);
            edge_mix<T>(at, PASS == kRows ? 0 : kEdgeStage, w8, st.acc + 4);
            __builtin_amdgcn_sched_barrier(0);
            range_update<T>(st, u8);
            edge_mix<T>(at, 0, u8, st.acc);
        }
        wave_lds_order();
    }
    if constexpr (TEAM) {
        // waves 2, 3 into 0, 1, then 1 into 0: two states fit the team's memory
        __shared__ uint32_t odd;
        float* area = reinterpret_cast<float*>(&lds_all[0]) + (wave & 1) * state_floats<PASS>();
        __syncthreads();
        if (wave >= 2) publish(st, area, lane);
        __syncthreads();
        if (wave < 2) absorb(st, area, lane);
        __syncthreads();
        if (wave == 1) publish(st, area, lane);
        __syncthreads();
        if (wave == 0) {
            absorb(st, area + state_floats<PASS>(), lane);
            edge_finish<T, PASS>(p, st, L.x1, w, (int)h, lane);
            const bool any = odd_state(st);
            if (lane == 0) odd = any;
        }
        __syncthreads();
        if (odd)
            slow_window<T, PASS>(p, w, (int)h, kEdgeWaves,
                                 [&](int k) { return (int32_t)(item - wave) + k; }, lds_all[0].pos);
    } else {
        const bool any = odd_state(st);
        if (lane == 0) p.odd[item * H + h] = any && slot < 0;
        if (slot >= 0) {   // a segment: its sums wait for edge_tail_kernel
            publish(st, p.partials + ((int64_t)slot * H + h) * state_floats<PASS>(), lane);
            if (h == 0 && lane == 0) p.slot_item[slot] = (int32_t)item;
        } else {
            edge_finish<T, PASS>(p, st, L.x1, w, (int)h, lane);
        }
    }
}

// What follows a pass of windows on single waves, one launch of workgroups for each:
// split windows, their segments joined in order (num_split x H); dslope[h] = -sum of
// the windows' shares of the rows' pass, in one fixed order (H, columns' pass with
// positions); the windows whose sums were not finite.
template <typename T, int PASS>
__global__ void __launch_bounds__(kWave * kEdgeWaves) edge_tail_kernel(const EdgeParams p)
{
    __shared__ __align__(16) _Float16 stage[16 * kHeadHalves];
    __shared__ float lds[16];
    __shared__ uint32_t odd;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const uint32_t H = (uint32_t)p.H, joins = (uint32_t)p.num_split * H;
    const uint32_t sums = PASS == kColumns && p.dims ? H : 0;
    if (blockIdx.x < joins) {
        const uint32_t h = blockIdx.x % H;
        const SplitInfo si = p.splits[blockIdx.x / H];
        if (wave == 0) {
            EdgeState<PASS> st;
            clear(st);
            for (int32_t k = 0; k < si.nseg; ++k)
                absorb(st, p.partials + ((int64_t)(si.first_slot + k) * H + h) * state_floats<PASS>(),
                       lane);
            edge_finish<T, PASS>(p, st, stage, si.w, (int)h, lane);
            const bool any = odd_state(st);
            if (lane == 0) odd = any;
        }
        __syncthreads();
        if (odd)
            slow_window<T, PASS>(p, si.w, (int)h, si.nseg,
                                 [&](int k) { return p.slot_item[si.first_slot + k]; }, lds);
        return;
    }
    if (blockIdx.x < joins + sums) {
        const uint32_t h = blockIdx.x - joins;
        sum_slopes<kWave * kEdgeWaves>(p.slope_parts + (int64_t)h * p.slope_windows, p.slope_windows,
                                       p.dslopes + h);
        return;
    }
    const int64_t units = p.num_items * H, groups = gridDim.x - joins - sums;
    for (int64_t base = (int64_t)(blockIdx.x - joins - sums) * kWave; base < units;
         base += groups * kWave) {
        uint64_t flagged = __ballot(base + lane < units && p.odd[min(base + lane, units - 1)] != 0u);
        for (; flagged; flagged &= flagged - 1) {   // (the same for every wave)
            const int64_t at = base + __builtin_ctzll(flagged);
            const int32_t item = (int32_t)(at / H);
            slow_window<T, PASS>(p, p.items[item].w, (int)(at % H), 1, [&](int) { return item; }, lds);
        }
    }
}

// dslopes without a launch to go with (teams, no nodes).
__global__ void __launch_bounds__(1024)
edge_slope_kernel(const float* __restrict__ parts, int32_t W, float* __restrict__ dslopes)
{
    sum_slopes<1024>(parts + (int64_t)blockIdx.x * W, W, dslopes + blockIdx.x);
}

__global__ void warm_edge_kernel() {}

hipError_t warm_edge(hipStream_t s)
{
    hipLaunchKernelGGL(warm_edge_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

constexpr int32_t kEdgeScanGroups = 1024;

template <typename T, int PASS, bool WIDE>
static void launch_edge(const EdgeParams& p, hipStream_t st)
{
    const dim3 block(kEdgeWaves * kWave);
    if (p.team > 1) {
        hipLaunchKernelGGL((edge_kernel<T, PASS, WIDE, true>),
                           dim3((unsigned)(p.num_items / kTeamSmall * p.H)), block, 0, st, p);
        return;
    }
    const int64_t groups = kXcds * ceil_div(ceil_div(p.num_items, kXcds) * p.H, kEdgeWaves);
    hipLaunchKernelGGL((edge_kernel<T, PASS, WIDE, false>), dim3((unsigned)groups), block, 0, st, p);
    const int64_t scans =
        std::min<int64_t>(kEdgeScanGroups, ceil_div(p.num_items * p.H, kWave));
    const int64_t sums = PASS == kColumns && p.dims ? p.H : 0;
    hipLaunchKernelGGL((edge_tail_kernel<T, PASS>), dim3((unsigned)(p.num_split * p.H + sums + scans)),
                       block, 0, st, p);
}

// Workspace of a pass: the marks of its units, its segments' items and sums.
struct EdgeSpace {
    size_t items = 0, partials = 0, bytes = 0;
};
static EdgeSpace edge_space(const f3s_plan* plan, bool backward)
{
    EdgeSpace s;   // (teams merge in LDS)
    const f3s_item_set& set = plan->masked;
    if (set.team == 1) {
        s.items = round_up(sizeof(uint32_t) * (size_t)set.num_items * plan->H);
        s.partials = s.items + round_up(sizeof(int32_t) * (size_t)set.num_slots);
        s.bytes = s.partials +
                  round_up(sizeof(float) *
                           (size_t)(backward ? state_floats<kRows>() : state_floats<kForward>()) *
                           plan->H * (size_t)set.num_slots);
    }
    return s;
}

template <int PASS>
static f3s_status launch_edge_pass(EdgeParams p, const f3s_plan* plan, int32_t dtype, char* ws,
                                   hipStream_t st)
{
    const f3s_item_set& set = plan->masked;
    const EdgeSpace space = edge_space(plan, PASS != kForward);
    p.odd = reinterpret_cast<uint32_t*>(ws);
    p.slot_item = reinterpret_cast<int32_t*>(ws + space.items);
    p.partials = reinterpret_cast<float*>(ws + space.partials);
    p.items = reinterpret_cast<const Item*>(set.items.ptr);
    p.num_items = set.num_items;
    p.splits = reinterpret_cast<const SplitInfo*>(set.splits.ptr);
    p.num_split = set.num_split;
    p.team = set.team;
    p.chunk_base = reinterpret_cast<const int32_t*>(plan->chunk_base.ptr);
    p.columns = reinterpret_cast<const uint32_t*>(plan->columns.ptr);
    p.W = plan->W;
    p.H = plan->H;
    p.xcd_contiguous = plan->xcd_contiguous;
    const bool nodes = wide_features(p.n, p.H);
    p.ref_shift = nodes ? 0 : 7;
    p.ref_magic = nodes ? 1u << 31 : (uint32_t)ceil_div((int64_t)1 << 31, p.H);
    p.no_ref = nodes ? kNoIdx : kNoRow;
    if (p.num_items <= 0) return F3S_OK;
    F3S_REQUIRE((p.num_items + p.num_split) * p.H < ((int64_t)1 << 24) * 3 &&   // (a grid's threads)
                    (p.num_split + 1) * p.H < ((int64_t)1 << 23) &&
                    (set.team == 1 || set.team == kTeamSmall),
                "edge attention: too many work items");
    // Offsets of 32 bits where every streamed tensor ends below kNoRow.
    const int64_t head = (int64_t)p.H * kEdgeHeadBytes;
    auto end = [&](const EdgeRows& x) { return (int64_t)(p.n - 1) * (int64_t)x.stride + head; };
    const bool wide = end(p.x1) > (int64_t)kNoRow || end(p.x2) > (int64_t)kNoRow;
    if (!wide) {
        p.x1.bytes = (uint32_t)end(p.x1);
        p.x2.bytes = (uint32_t)end(p.x2);
    }
    if (dtype == F3S_F16) {
        if (wide) launch_edge<_Float16, PASS, true>(p, st);
        else launch_edge<_Float16, PASS, false>(p, st);
    } else {
        if (wide) launch_edge<__bf16, PASS, true>(p, st);
        else launch_edge<__bf16, PASS, false>(p, st);
    }
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

static f3s_status check_edge(const f3s_plan* plan, int32_t dtype, int32_t n, int32_t H, float cap,
                             const float* positions, int32_t dims, const float* slopes,
                             const char* who)
{
    if (n < 0 || (dtype != F3S_F16 && dtype != F3S_BF16)) {
        set_error(std::string(who) + ": negative n or unknown dtype");
        return F3S_EINVAL;
    }
    if (!(cap == 0.f || (cap > 1e-30f && cap < 1e30f)) || dims < 0 || dims > 3 ||
        (dims > 0 && (!slopes || (n > 0 && !positions)))) {
        set_error(std::string(who) + ": cap is 0 (none) or from 1e-30 to 1e30, positions have "
                                     "1 to 3 dims (0: none) and slopes");
        return F3S_EINVAL;
    }
    if (!plan || plan->compiled_n < 0 || plan->compiled_n != n || plan->H != H) {
        set_error(std::string(who) + ": needs a plan compiled for this n and H");
        return F3S_EINVAL;
    }
    return F3S_OK;
}

// Rows at 16-byte boundaries, wide enough for the heads.
static bool edge_rows_ok(const void* ptr, int64_t stride, int32_t H)
{
    return ptr && ((uintptr_t)ptr & 15) == 0 && stride % 8 == 0 && stride >= (int64_t)H * kD &&
           stride < ((int64_t)1 << 30);
}

static EdgeParams edge_params(int32_t n, float scale, float cap, const float* positions, int32_t dims,
                              const float* slopes)
{
    EdgeParams p{};
    p.n = n;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.cap = cap;
    p.cap_in = cap > 0.f ? std::clamp(scale / cap, -FLT_MAX, FLT_MAX) : 0.f;   // (0 x inf)
    p.cap_log2 = cap * kLog2e;
    p.positions = positions;
    p.dims = dims;
    p.stat_words = stat_words(dims);
    p.slopes = slopes;
    return p;
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_edge_attention_workspace(const f3s_plan* plan, const f3s_plan* reversed,
                                        int32_t dims, int64_t* bytes)
{
    F3S_REQUIRE(plan && bytes && dims >= 0 && dims <= 3,
                "f3s_edge_attention_workspace: NULL pointer, or dims not 0 to 3");
    size_t need = edge_space(plan, reversed != nullptr).bytes;
    if (reversed) {
        const size_t cells = (size_t)std::max(plan->compiled_n, 0) * plan->H;
        need = std::max(need, edge_space(reversed, true).bytes) + round_up(cells * 4 * stat_words(dims)) +
               round_up(sizeof(float) * (size_t)plan->W * plan->H);
    }
    *bytes = (int64_t)need;
    return F3S_OK;
}

f3s_status f3s_edge_attention_fwd(const f3s_plan* plan, const uint16_t* Q, int64_t q_stride,
                                  const uint16_t* K, int64_t k_stride, const uint16_t* V,
                                  int64_t v_stride, uint16_t* O, int64_t o_stride, float* lse,
                                  int32_t dtype, int32_t n, int32_t H, float scale, float cap,
                                  const float* positions, int32_t dims, const float* slopes,
                                  void* workspace, int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_edge(plan, dtype, n, H, cap, positions, dims, slopes, "f3s_edge_attention_fwd"));
    if (n == 0) return F3S_OK;
    F3S_REQUIRE(edge_rows_ok(Q, q_stride, H) && edge_rows_ok(K, k_stride, H) &&
                    edge_rows_ok(V, v_stride, H) && edge_rows_ok(O, o_stride, H),
                "f3s_edge_attention_fwd: NULL or misaligned pointer, or a row stride that is no "
                "multiple of 8 or below H * 64");
    const int64_t need = (int64_t)edge_space(plan, false).bytes;
    F3S_REQUIRE(workspace_bytes >= need && (workspace || need == 0) &&
                    ((uintptr_t)workspace & 15) == 0,
                "f3s_edge_attention_fwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    EdgeParams p = edge_params(n, scale, cap, positions, dims, slopes);
    p.x1 = rows_of(K, k_stride);
    p.x2 = rows_of(V, v_stride);
    p.own1 = rows_of(Q, q_stride);
    p.out1 = rows_of(O, o_stride);
    p.lse = lse;
    return launch_edge_pass<kForward>(p, plan, dtype, static_cast<char*>(workspace),
                                      as_stream(stream));
}

f3s_status f3s_edge_attention_bwd(const f3s_plan* plan, const f3s_plan* reversed, const uint16_t* Q,
                                  int64_t q_stride, const uint16_t* K, int64_t k_stride,
                                  const uint16_t* V, int64_t v_stride, const float* lse,
                                  const uint16_t* dO, int64_t do_stride, uint16_t* dQ,
                                  int64_t dq_stride, uint16_t* dK, int64_t dk_stride, uint16_t* dV,
                                  int64_t dv_stride, float* dslopes, int32_t dtype, int32_t n,
                                  int32_t H, float scale, float cap, const float* positions,
                                  int32_t dims, const float* slopes, void* workspace,
                                  int64_t workspace_bytes, void* stream)
{
    F3S_TRY(check_edge(plan, dtype, n, H, cap, positions, dims, slopes, "f3s_edge_attention_bwd"));
    F3S_TRY(check_edge(reversed, dtype, n, H, cap, positions, dims, slopes,
                       "f3s_edge_attention_bwd (reversed)"));
    F3S_REQUIRE(dims == 0 || dslopes, "f3s_edge_attention_bwd: NULL pointer");
    F3S_REQUIRE(n == 0 || (edge_rows_ok(Q, q_stride, H) && edge_rows_ok(K, k_stride, H) &&
                           edge_rows_ok(V, v_stride, H) && edge_rows_ok(dO, do_stride, H) &&
                           edge_rows_ok(dQ, dq_stride, H) && edge_rows_ok(dK, dk_stride, H) &&
                           edge_rows_ok(dV, dv_stride, H) && lse),
                "f3s_edge_attention_bwd: NULL or misaligned pointer, or a row stride that is no "
                "multiple of 8 or below H * 64");
    int64_t need = 0;
    F3S_TRY(f3s_edge_attention_workspace(plan, reversed, dims, &need));
    F3S_REQUIRE(workspace_bytes >= need && (workspace || need == 0) &&
                    ((uintptr_t)workspace & 15) == 0,
                "f3s_edge_attention_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    EdgeParams p = edge_params(n, scale, cap, positions, dims, slopes);
    if (n > 0) {
        char* ws = static_cast<char*>(workspace);
        p.stats = reinterpret_cast<float*>(ws);
        ws += round_up((size_t)n * H * 4 * p.stat_words);
        p.slope_parts = reinterpret_cast<float*>(ws);
        ws += round_up(sizeof(float) * (size_t)plan->W * H);
        p.slope_windows = plan->W;
        p.dslopes = dslopes;
        p.lse = const_cast<float*>(lse);
        EdgeParams rows = p;
        rows.x1 = rows_of(K, k_stride);
        rows.x2 = rows_of(V, v_stride);
        rows.own1 = rows_of(Q, q_stride);
        rows.own2 = rows_of(dO, do_stride);
        rows.out1 = rows_of(dQ, dq_stride);
        F3S_TRY(launch_edge_pass<kRows>(rows, plan, dtype, ws, st));
        EdgeParams cols = p;
        cols.x1 = rows_of(Q, q_stride);
        cols.x2 = rows_of(dO, do_stride);
        cols.own1 = rows_of(K, k_stride);
        cols.own2 = rows_of(V, v_stride);
        cols.out1 = rows_of(dK, dk_stride);
        cols.out2 = rows_of(dV, dv_stride);
        F3S_TRY(launch_edge_pass<kColumns>(cols, reversed, dtype, ws, st));
    }
    if (dims > 0 && (n == 0 || reversed->masked.team > 1))
        hipLaunchKernelGGL(edge_slope_kernel, dim3((unsigned)H), dim3(1024), 0, st, p.slope_parts,
                           n > 0 ? plan->W : 0, dslopes);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

}  // extern "C"
