// diff_attention.hip -- differential attention over a graph's edges, and its
// gradient, on the compiled column lists of a plan (attention.hip).
//
// Per head two maps of 64 dims (q = [q1 q2], k = [k1 k2]) and values of 128:
//   p_c(i, j) = softmax over the edges i -> j of scale q_c(i).k_c(j)
//   o(i) = sum_j (p_1 - lam p_2)(i, j) v(j)           (rows without edges: 0)
// and, for a gradient do(i), with g = do(i).v(j) and D_c(i) = sum_j p_c g,
//   ds_1 = p_1 (g - D_1),  ds_2 = -lam p_2 (g - D_2)
//   dq_c(i) = scale sum_j ds_c k_c(j),  dk_c(j) = scale sum_i ds_c q_c(i)
//   dv(j) = sum_i (p_1 - lam p_2) do(i),  dlam = -sum_i D_2(i)
//
// Three passes of one shape: a wave takes a window of 16 rows of one head and
// streams the rows at the other ends of its edges past it, 32 per chunk, two
// 256-byte rows each:
//   forward  k, v past q:            m, l and the sums of p_1 v, p_2 v
//   rows     k, v past q, do:        the sums of p_c g k_c, p_c k_c and p_c g:
//            dq_c = scale (sum p_c g k_c - D_c sum p_c k_c) needs no second
//            sweep for D, and nothing of o is kept from the forward pass but
//            log-sum-exps
//   columns  q, do past k, v, on the plan of the reversed edges: dk, dv; no
//            atomics, so gradients are the same from run to run
// What bounds them is the random 512 bytes per edge and head; the matrix cores
// work on 16 x 32 pairs of which a sparse window uses about one in 16.
//
// Every 16-bit weight (p, p g, ds) is the sum of two (split8), two MFMAs
// instead of one: p_1 and p_2 nearly cancel where lam is near 1 and the maps
// are alike, and what a single rounding of each leaves is then large beside
// their difference.  binary16's two halves end at 2^-25, so what can be far below 1
// is scaled: p g and ds by a power of two per row that follows them
// (range_update), p of the rows and p_1 - lam p_2 of the columns by a fixed 2^14
// (kLift).  Sums and softmax statistics are in float32.
//
// A value that is infinite or NaN reaches, through the matrix cores, rows of its
// window that have no edge to it (0 x inf).  So a window whose sums are not
// finite at the end is done twice more: once to mark the sums that have such a
// value on an edge of theirs, which become NaN, and once without those values.
// Large graphs leave that to a second launch, which finds nothing as a rule: in
// the pass itself its registers would be taken from the loads in flight.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstddef>

#include "attn_plan.hpp"
#include "half_types.hpp"

namespace f3s {

constexpr int kMapD = 64;                  // dims of one map
constexpr int kHeadD = 2 * kMapD;          // q, k, v, o of one head
constexpr int kHeadBytes = kHeadD * 2;
// A chunk's rows in LDS, 256 bytes each, a row's 16-byte pieces in an order of its
// own (piece p at p ^ kSwizzle(row)): 16 rows' pieces of one number, which the
// products with the window's rows read, and four rows' pairs of pieces, which the
// transposing reads take, then lie in distinct banks without padding.
constexpr int kRowHalves = kHeadD;
__device__ __forceinline__ int swizzle(int row) { return ((row & 7) << 1) | ((row >> 3) & 1); }

// The lane again, for the compiler a new value: what is derived from it is then made
// where it is used and not held in registers through the chunk loop.
__device__ __forceinline__ int anew(int lane)
{
    asm volatile("" : "+v"(lane));
    return lane;
}

enum DiffPass : int { kDiffForward = 0, kDiffRows = 1, kDiffColumns = 2 };

// Rows r of a tensor start `stride` bytes apart; a head's 256 bytes are
// contiguous, heads adjacent.
struct DiffRows {
    const char* ptr;
    uint64_t stride;
    uint32_t bytes;   // narrow launches: end of the last row (loads past it read 0)
};

struct DiffParams {
    DiffRows x1, x2;        // streamed: k and v; q and do on the reversed edges
    DiffRows own1, own2;    // the window's own rows: q and do; k and v
    DiffRows out1, out2;    // o; dq; dk and dv
    const float* lam;       // [H]
    float* lse;             // [n][H][2], log2; forward: written (NULL: not)
    float* stats;           // [n][H][4]: lse_1, lse_2, D_1, D_2
    uint32_t stats_bytes;
    float* dlam_parts;      // [H][W]
    const Item* items;
    const int32_t* chunk_base;
    const uint32_t* columns;
    const SplitInfo* splits;
    float* partials;
    int64_t num_items, num_split;
    int32_t W, n, H;
    int32_t xcd_contiguous;
    // the lists' references: node indices, or node * H * 128 (below kNoRow);
    // node = ((ref >> shift) * magic) >> 31, magic 2^31 or ceil(2^31 / H), which is
    // exact below 2^25
    uint32_t ref_shift, ref_magic, no_ref;
    uint32_t* queue;        // next unit of each XCD's share, kQueueStride apart; NULL: a unit
                            // per wave
    uint32_t* odd;          // [items][H]: sums that are not finite (kDiffMain writes,
                            // kDiffRepair reads)
    float scale, scale_log2;
};

// A wave's sums: 16 tiles of 16 dims, lane (g, r) holding dims 16 t + 4 g + v of
// row r in tile t of its eight (v: the element).
//   forward: tiles 0-7 of map 1 and 8-15 of map 2, scaled by 2^-x, x the running
//            maxima; y: l
//   rows:    4 m + t: sum p g k of map m, scaled by 2^-x[m]; 8 + 4 m + t: sum p k;
//            y: sum p g, z: sum p
//   columns: 4 m + t: sum ds q of map m, scaled by 2^-x[m]; 8 + t: dv
struct DiffState {
    f4 acc[16];
    float x[2], y[2], z[2];
};
constexpr int kDiffPartial = 18 * kWave * 4;   // floats of a published state

// First tile and number of tiles that x[c] scales.
template <int PASS>
struct Scaled {
    static constexpr int count = PASS == kDiffForward ? 8 : 4;
    static constexpr int first(int c) { return count * c; }
};

__device__ __forceinline__ void clear(DiffState& s)
{
#pragma unroll
    for (int t = 0; t < 16; ++t) s.acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    s.x[0] = s.x[1] = -INFINITY;
    s.y[0] = s.y[1] = s.z[0] = s.z[1] = 0.f;
}

template <int PASS>
__device__ __forceinline__ void rescale(DiffState& s, int c, float factor)
{
#pragma unroll
    for (int t = 0; t < Scaled<PASS>::count; ++t) s.acc[Scaled<PASS>::first(c) + t] *= factor;
}

__device__ __forceinline__ void publish(const DiffState& s, float* dst, int lane)
{
#pragma unroll
    for (int t = 0; t < 16; ++t) *reinterpret_cast<f4*>(&dst[(t * kWave + lane) * 4]) = s.acc[t];
    *reinterpret_cast<f4*>(&dst[(16 * kWave + lane) * 4]) = f4{s.x[0], s.x[1], s.y[0], s.y[1]};
    *reinterpret_cast<f4*>(&dst[(17 * kWave + lane) * 4]) = f4{s.z[0], s.z[1], 0.f, 0.f};
}

// Takes a published state into s.
template <int PASS>
__device__ __forceinline__ void absorb(DiffState& s, const float* src, int lane)
{
    const f4 xy = *reinterpret_cast<const f4*>(&src[(16 * kWave + lane) * 4]);
    const f4 z = *reinterpret_cast<const f4*>(&src[(17 * kWave + lane) * 4]);
    f4 a[16];   // (all on their way before the first is waited for)
#pragma unroll
    for (int t = 0; t < 16; ++t)
        a[t] = *reinterpret_cast<const f4*>(&src[(t * kWave + lane) * 4]);
    __builtin_amdgcn_sched_barrier(0);
    float theirs[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const float top = __builtin_fmaxf(s.x[c], xy[c]);
        const float mine = top == -INFINITY ? 0.f : fast_exp2(s.x[c] - top);
        theirs[c] = top == -INFINITY ? 0.f : fast_exp2(xy[c] - top);
        rescale<PASS>(s, c, mine);
        if constexpr (PASS == kDiffForward)
            s.y[c] = s.y[c] * mine + xy[2 + c] * theirs[c];
        else
            s.y[c] += xy[2 + c];
        s.z[c] += z[c];
        s.x[c] = top;
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const int c = t / Scaled<PASS>::count;
        s.acc[t] += c < 2 ? a[t] * theirs[c] : a[t];
    }
}

// One chunk's slots of a record: byte offsets into x1 and x2 (narrow) or node
// indices (wide), row masks, and byte offsets into stats.
struct DiffRecord {
    uint32_t at1[kChunk], at2[kChunk], rm[kChunk], st[kChunk];
};
constexpr int kBlockRecs = 2;   // records read, converted and handed out together
static_assert(kBlockRecs * 2 * kChunk == 2 * kWave, "two words per lane");
struct __align__(256) DiffLds {
    _Float16 x1[kChunk * kRowHalves];
    _Float16 x2[kChunk * kRowHalves];
    DiffRecord rec[2 * kBlockRecs];
    float stats[kChunk * 4];
};
static_assert(sizeof(DiffLds) >= sizeof(float) * kDiffPartial,
              "a published state fits a wave's memory");

template <typename T, bool WIDE>
__device__ __forceinline__ typename Half<T>::v8 diff_load(__amdgpu_buffer_rsrc_t rs,
                                                          const DiffRows& x, uint32_t at,
                                                          uint32_t extra)
{
    if constexpr (!WIDE) {
        return __builtin_bit_cast(typename Half<T>::v8,
                                  __builtin_amdgcn_raw_buffer_load_b128(rs, at + extra, 0, 0));
    } else {
        typename Half<T>::v8 v = {};
        if (at != kNoIdx)
            v = *reinterpret_cast<const typename Half<T>::v8*>(x.ptr + at * x.stride + extra);
        return v;
    }
}

typedef __attribute__((address_space(3))) char* LdsPtr;
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at)
{
    return *(__attribute__((address_space(3))) V*)(LdsPtr)(uintptr_t)at;
}
template <typename V>
__device__ __forceinline__ void lds_write(uint32_t at, V v)
{
    *(__attribute__((address_space(3))) V*)(LdsPtr)(uintptr_t)at = v;
}

// Where a lane reads and writes in a stage (addresses in LDS).  A piece's place
// is an exclusive or of the row's and the piece's number, so the addresses of all
// pieces come from one by exclusive or with constants, made where they are used
// (held in registers, they would be some forty of them; `held` keeps the compiler
// from that).
struct Places {
    uint32_t row;     // piece g of row r
    uint32_t column;  // what lane r of group g hands the transposing read of tile 0
    uint32_t write;   // piece r of row g
};
__device__ __forceinline__ Places places(const _Float16* stage, int lane)
{
    const int g = lane >> 4, r = lane & 15, i = r >> 2, c = r & 3;
    const uint32_t base = (uint32_t)(uintptr_t)(LdsPtr)stage;
    return Places{base + 256 * r + 16 * (g ^ swizzle(r)),
                  base + 256 * (4 * g + i) + 16 * ((c >> 1) ^ swizzle(4 * g + i)) + 8 * (c & 1),
                  base + 256 * g + 16 * (r ^ swizzle(g))};
}
__device__ __forceinline__ void held(Places& p)
{
    asm volatile("" : "+v"(p.row), "+v"(p.column), "+v"(p.write));
}
constexpr uint32_t kStageBytes = sizeof(_Float16) * kChunk * kRowHalves;   // x2 after x1
constexpr uint32_t kHalfStage = kStageBytes / 2;                          // 16 rows

// Rows 4 i + g, i = 0 .. 7, from the lane's pieces (number r of each).
template <typename V>
__device__ __forceinline__ void write_rows(const Places& p, uint32_t stage, const V (&x)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        lds_write(((p.write ^ (128 * (i & 1) + 16 * ((i >> 1) & 1))) + stage) + 1024 * i, x[i]);
}

// The 16 dims from 16 t of the chunk's slots as an A operand: lane (g, r) gets
// dim 16 t + r of its eight slots (slot_of).  Each group of 16 lanes hands four
// rows of 16 values to the transposing read, lane r its piece of row r / 4, and
// receives column r of them; twice, for slots 4 g .. and 16 + 4 g ...
template <typename T>
__device__ __forceinline__ typename Half<T>::v8 transposed(const Places& p, uint32_t stage, int t)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* lds4;
    const uint32_t at = (p.column ^ (32 * t)) + stage;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)at);
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(at + kHalfStage));
    return __builtin_bit_cast(typename Half<T>::v8,
                              s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// acc[t] += sum over the chunk's slots of w (the lane's slots of row r) times the
// 16 dims of tile t0 + t, N tiles x.  (Products of one sum are N apart: they need
// not wait for each other.)
template <typename T, int N = 4>
struct Tiles {
    typename Half<T>::v8 x[N];
    __device__ __forceinline__ Tiles(const Places& p, uint32_t stage, int t0)
    {
#pragma unroll
        for (int t = 0; t < N; ++t) x[t] = transposed<T>(p, stage, t0 + t);
    }
    __device__ __forceinline__ void mix(const typename Half<T>::v8& hi,
                                        const typename Half<T>::v8& lo, f4* acc) const
    {
#pragma unroll
        for (int t = 0; t < N; ++t) acc[t] = Half<T>::mfma(x[t], hi, acc[t]);
#pragma unroll
        for (int t = 0; t < N; ++t) acc[t] = Half<T>::mfma(x[t], lo, acc[t]);
    }
    __device__ __forceinline__ void mix(const float (&w)[8], f4* acc) const
    {
        typename Half<T>::v8 hi, lo;
        split8<T>(w, hi, lo);
        mix(hi, lo, acc);
    }
};

// 16 rows of a stage times the window's rows, dims 32 (f0 + f) .., NF of them.
template <typename T, int NF>
__device__ __forceinline__ f4 products(const Places& p, uint32_t stage, int f0,
                                       const typename Half<T>::v8 (&own)[4])
{
    f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = f0; f < f0 + NF; ++f)
        s = Half<T>::mfma(lds_read<typename Half<T>::v8>((p.row ^ (64 * f)) + stage), own[f], s);
    return s;
}

// A staged chunk's values, to stage `to`: MARK: 1 where infinite or NaN, else 0;
// CLEAN: 0 there.
enum Sweep : int { kSweepPlain = 0, kSweepMark = 1, kSweepClean = 2 };
template <typename T>
__device__ __forceinline__ void replace_odd(const Places& p, uint32_t stage, uint32_t to, int sweep)
{
    typedef typename Half<T>::v8 v8;
    wave_lds_order();   // its readers so far are done
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        const uint32_t at = ((p.write ^ (128 * (i & 1) + 16 * ((i >> 1) & 1))) + stage) + 1024 * i;
        v8 x = lds_read<v8>(at);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = (float)x[k];
            const bool odd = !(f - f == 0.f);
            x[k] = sweep == kSweepMark ? (T)(odd ? 1.f : 0.f) : odd ? (T)0.f : x[k];
        }
        lds_write(at - stage + to, x);
    }
    wave_lds_order();
}

// Which of the lane's eight slots row r attends: all bits or none.
typedef uint32_t Attends[8];
__device__ __forceinline__ float where(uint32_t on, float x, float other)
{
    return __uint_as_float((__float_as_uint(x) & on) | (__float_as_uint(other) & ~on));
}
__device__ __forceinline__ float where(uint32_t on, float x)
{
    return __uint_as_float(__float_as_uint(x) & on);
}

// From a record's masks at `masks`, anew wherever they are used: two LDS reads,
// where eight registers would be held.
__device__ __forceinline__ void attends(uint32_t masks, int lane, Attends& on)
{
    const int l = anew(lane), r = l & 15, rbit = (r & 1) ? 16 + (r >> 1) : (r >> 1);
    const uint32_t at = masks + 16 * (l >> 4);   // slots 4 g .. and 16 + 4 g ..
    const u4 a = lds_read<u4>(at), b = lds_read<u4>(at + 64);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        on[j] = (uint32_t)__builtin_amdgcn_sbfe((int)(j < 4 ? a[j & 3] : b[j & 3]), rbit, 1);
}

template <int N>
__device__ __forceinline__ void edge_weights(float (&w)[N][8], const Attends& on)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = where(on[j], 1.f);
}

// One map's softmax step (log2): x = s c, c > 0; the running maximum is moved when
// a chunk's exceeds it by more than kLazy.  p[j] = 2^(x - m), 0 where not attended;
// y is the lane's share of l.
__device__ __forceinline__ void map_update(DiffState& st, int m, const f4 s0, const f4 s1,
                                           const Attends& on, float c, float (&p)[8])
{
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = where(on[j], j < 4 ? s0[j & 3] : s1[j & 3], -INFINITY);
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = __builtin_fmaxf(top, s[j]);
    top = row_max4(top) * c;
    if (__ballot(top > st.x[m] + kLazy)) {
        if (top > st.x[m] + kLazy) {
            const float corr = fast_exp2(st.x[m] - top);
            st.y[m] *= corr;
            rescale<kDiffForward>(st, m, corr);
            st.x[m] = top;
        }
    }
    const float mu = st.x[m] == -INFINITY ? 0.f : st.x[m];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = fast_exp2(__builtin_fmaf(s[j], c, -mu));
        st.y[m] += p[j];
    }
}

// Weights of a size of 1 at most, in binary16: with |w| <= 2 they stay below 2^15, and
// their halves end at 2^-39.  (A node that a row hardly attends, or that only rows of
// very many edges do, has weights of 2^-17 and less alone: unscaled, 2^-20 was off by
// 2^-6 of itself.)
// (In the rows' pass as an addend of the exponent: all its sums are divided by the
// weights' own.  A row of 10^5 equal edges has weights of 2^-17, all rounded the same
// way: dq, a difference of two sums of them, was off by 2^-8 of either.)
template <typename T>
constexpr float kLift = Half<T>::kRange ? 16384.f : 1.f;
template <typename T>
constexpr float kLiftLog2 = Half<T>::kRange ? 14.f : 0.f;
// Such a weight's exponent.  A weight is at most 1, but for what a log-sum-exp of 24
// bits leaves (logits past 2^24 come out as 2^2 and more): kept at 2 (rows, lifted) and
// at 1 (columns), inside the type.  NaN stays.
template <typename T>
__device__ __forceinline__ float lifted(float x, float most)
{
    return Half<T>::kRange ? __builtin_elementwise_minimum(x, most) : x;
}

// Scales weights of unknown size into binary16: a power of two per row, st.x[m],
// moved (and the sums that it scales with it) when a weight would come within a
// factor of four of the type's end, to put that weight at 2^3 to 2^4.
template <typename T>
__device__ __forceinline__ void range_update(DiffState& st, int m, float (&w)[8])
{
    if constexpr (Half<T>::kRange) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(w[j]));
        most = row_max4(most);
        // (2^x may be far below 2^-126: compare exponents)
        const float e = most > 0.f ? (float)__builtin_amdgcn_frexp_expf(most) : -INFINITY;
        if (__ballot(e > st.x[m] + 14.f)) {
            if (e > st.x[m] + 14.f) {
                const float x = __builtin_fminf(e, 128.f) - 4.f;
                rescale<kDiffRows>(st, m, fast_exp2(st.x[m] - x));
                st.x[m] = x;
            }
        }
        const int f = st.x[m] == -INFINITY ? 0 : (int)-st.x[m];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_ldexpf(w[j], f);
    }
}

// Rows of 128 values leave whole, through a stage: val(t) is the lane's part of
// tile t, dims 16 t + 4 g .. + 3.
template <typename T, typename F>
__device__ __forceinline__ void store_rows(const DiffRows& out, _Float16* stage, int32_t w,
                                           int32_t n, uint32_t head_off, int lane, F val)
{
    typedef typename Half<T>::v8 v8;
    typedef typename Half<T>::v4 v4;
    const int g = lane >> 4, r = lane & 15;
#pragma unroll
    for (int t = 0; t < 8; ++t)
        *reinterpret_cast<v4*>(&stage[r * kRowHalves + 8 * ((2 * t + (g >> 1)) ^ swizzle(r)) +
                                      4 * (g & 1)]) = __builtin_convertvector(val(t), v4);
    wave_lds_order();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int rr = 4 * v + g;
        const v8 x = *reinterpret_cast<const v8*>(&stage[rr * kRowHalves + 8 * (r ^ swizzle(rr))]);
        const int32_t row = w * 16 + rr;
        if (row < n)
            *reinterpret_cast<v8*>(const_cast<char*>(out.ptr) + row * out.stride + head_off +
                                   16 * r) = x;
    }
    wave_lds_order();
}

__device__ __forceinline__ float over_groups(float x)
{
    x += __shfl_xor(x, 16, kWave);
    return x + __shfl_xor(x, 32, kWave);
}

// A window's results from its sums.  `stage`: 2 x 16 rows.
template <typename T, int PASS>
__device__ __forceinline__ void diff_finish(const DiffParams& p, DiffState& st, _Float16* stage,
                                            int32_t w, int h, float lam, int lane)
{
    lane = anew(lane);
    const int g = lane >> 4, r = lane & 15;
    const int32_t row = w * 16 + r;
    const uint32_t head_off = (uint32_t)h * kHeadBytes;
    if constexpr (PASS == kDiffForward) {
        const float l1 = over_groups(st.y[0]), l2 = over_groups(st.y[1]);
        // (a row of NaN is some; one map's logits all -inf: 0 / 0)
        const bool some = l1 != 0.f || l2 != 0.f;
        const float f1 = some ? 1.f / l1 : 0.f, f2 = some ? lam / l2 : 0.f;
        store_rows<T>(p.out1, stage, w, p.n, head_off, lane, [&](int t) {
            const f4 o = st.acc[t] * f1 - st.acc[8 + t] * f2;
            return some ? o : f4{0.f, 0.f, 0.f, 0.f};
        });
        if (p.lse && g == 0 && row < p.n)
            *reinterpret_cast<float2*>(p.lse + ((int64_t)row * p.H + h) * 2) =
                some ? make_float2(st.x[0] + __log2f(l1), st.x[1] + __log2f(l2))
                     : make_float2(0.f, 0.f);
    } else if constexpr (PASS == kDiffRows) {
        // The weights' own sums (1, but for the rounding of the log-sum-exps)
        // divide: dlam is a sum over all rows, in which an error common to a
        // row's weights would not average out.
        const float l1 = over_groups(st.z[0]), l2 = over_groups(st.z[1]);
        const float i1 = l1 != 0.f ? 1.f / l1 : 0.f, i2 = l2 != 0.f ? 1.f / l2 : 0.f;
        const float sign = (r & 1) ? -1.f : 1.f;   // (of do in the sums)
        const float d1 = sign * over_groups(st.y[0]) * i1, d2 = sign * over_groups(st.y[1]) * i2;
        const float f1 = sign * fast_exp2(st.x[0]), f2 = sign * fast_exp2(st.x[1]);   // (0: unset)
        const float c1 = p.scale * i1, c2 = -lam * p.scale * i2;
        store_rows<T>(p.out1, stage, w, p.n, head_off, lane, [&](int t) {
            return t < 4 ? c1 * (st.acc[t] * f1 - d1 * st.acc[8 + t])
                         : c2 * (st.acc[t] * f2 - d2 * st.acc[8 + t]);
        });
        if (g == 0 && row < p.n)
            *reinterpret_cast<float2*>(p.stats + ((int64_t)row * p.H + h) * 4 + 2) =
                make_float2(d1, d2);
        // the window's share of dlam: rows 0 to 15 in one fixed order
        float s = row < p.n ? d2 : 0.f;
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor(s, off, kWave);
        if (lane == 0) p.dlam_parts[(int64_t)h * p.W + w] = s;
    } else {
        const float f1 = fast_exp2(st.x[0]), f2 = fast_exp2(st.x[1]);
        const float back =
            Half<T>::kRange ? __builtin_fmaxf(1.f, __builtin_fabsf(lam)) * (1.f / kLift<T>) : 1.f;
        store_rows<T>(p.out1, stage, w, p.n, head_off, lane, [&](int t) {
            return t < 4 ? p.scale * (st.acc[t] * f1) : -lam * p.scale * (st.acc[t] * f2);
        });
        store_rows<T>(p.out2, stage, w, p.n, head_off, lane,
                      [&](int t) { return st.acc[8 + t] * back; });
    }
}

constexpr int kDiffWaves = 4;   // per workgroup
static_assert(kDiffWaves == kTeamSmall, "a team fills its workgroup");

constexpr int kQueueStride = 64;   // words: a counter per cache line and more

// kDiffMain: a window (or segment) per wave, windows one after another; kDiffTeam:
// four waves share a window (small graphs); kDiffRepair: the windows that kDiffMain
// marked in p.odd.
enum DiffMode : int { kDiffMain = 0, kDiffTeam = 1, kDiffRepair = 2 };

// A wave's work: one item and head.  there: such an item is; w < 0: without a
// window; end: past the last one.
struct Unit {
    uint32_t item;
    int32_t w, slot, h, cb, ce;
    float lam;
    bool there, end;
};

__device__ __forceinline__ float uniform(float x)
{
    return __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(x)));
}

template <typename V>
__device__ __forceinline__ V scalar_load(const V* at)
{
    typedef const __attribute__((address_space(4))) V* Constant;
    return *(Constant)(uintptr_t)at;
}

// Large graphs' waves take unit after unit from a queue, their chunks one stream:
// the records, own rows and first chunk of a unit are loaded while the one before
// it is still being computed.  (A window has some 7 to 20 chunks; a wave of its
// own for each met three memory latencies before its first.  500,000 nodes, 6.5 M
// edges, microseconds, a wave per window -> queue: forward 452 -> 398, rows 774 ->
// 427, columns 626 -> 514; 100,000 nodes of communities, 4.1 M edges, two heads,
// bfloat16: 382 -> 323, 432 -> 399, 471 -> 439.  Part of it is that nothing is
// spilled any more: a reload in the chunk loop waits for every gather in flight.)
template <typename T, int PASS, bool WIDE, int MODE>
__global__ void __launch_bounds__(kWave * kDiffWaves) __attribute__((amdgpu_waves_per_eu(2)))
diff_kernel(const DiffParams p)
{
    typedef typename Half<T>::v8 v8;
    __shared__ DiffLds lds_all[kDiffWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    DiffLds& L = lds_all[wave];
    const uint32_t H = (uint32_t)p.H;
    const int32_t n = p.n;

    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(p.x1.ptr, p.x1.bytes);
    const __amdgpu_buffer_rsrc_t r2 = make_rsrc(p.x2.ptr, p.x2.bytes);
    const __amdgpu_buffer_rsrc_t rst = make_rsrc(p.stats, p.stats_bytes);

    // Unit `at` of share x.  A scheduled plan's items are eight interleaved shares,
    // share x for XCD x, and the dispatcher deals workgroups to the XCDs in turn:
    // workgroup b takes items of share b % 8, the heads of an item one after another.
    // A natural-order plan's shares are contiguous instead.
    const uint32_t xcd = blockIdx.x % kXcds;
    const uint32_t share = (uint32_t)((p.num_items + kXcds - 1) / kXcds);
    // By scalar loads (the lists are constant; a wave's vector registers are all in
    // use).  They are waited for with the next LDS access, so units are asked for
    // where a wave waits for memory anyway.
    auto unit = [&](uint32_t item, uint32_t h, bool there) __attribute__((always_inline)) -> Unit {
        there = there && item < (uint32_t)p.num_items;
        const uint32_t i = there ? item : 0;
        const u4 it = scalar_load(reinterpret_cast<const u4*>(p.items + i));
        Unit u;
        u.item = i;
        u.there = there;
        u.w = there && (int32_t)it[0] < p.W ? (int32_t)it[0] : -1;
        u.slot = (int32_t)it[3];
        u.h = (int32_t)h;
        u.cb = scalar_load(p.chunk_base + i);
        u.ce = u.w < 0 ? u.cb : scalar_load(p.chunk_base + i + 1);
        u.lam = scalar_load(p.lam + h);
        u.end = false;
        return u;
    };
    auto of_share = [&](uint32_t at) __attribute__((always_inline)) -> Unit {
        const uint32_t i = at / H;
        Unit u = unit(p.xcd_contiguous ? xcd * share + i : i * kXcds + xcd, at % H, i < share);
        u.end = i >= share;
        return u;
    };
    // The queue's next unit, asked for one unit ahead (one lane's atomic; every
    // wave ends once its unit is past the share, which the counter only moves to).
    auto ticket = [&]() __attribute__((always_inline)) -> uint32_t {
        uint32_t t = 0;
        if (p.queue && lane == 0) t = atomicAdd(p.queue + xcd * kQueueStride, 1u);
        return t;
    };
    auto redeem = [&](uint32_t t) __attribute__((always_inline)) -> Unit {
        return of_share(p.queue ? (uint32_t)__builtin_amdgcn_readfirstlane((int)t) : share * H);
    };

    // ---- the window's own rows, in operand order: dims 32 f + 8 g .. of row r
    // (rows past the last are not stored) ----
    auto own_load = [&](const DiffRows& x, const Unit& u, v8 (&f)[4]) __attribute__((always_inline)) {
        const int l = anew(lane);
        const int32_t row = min(max(u.w, 0) * 16 + (l & 15), n - 1);
        const char* src = x.ptr + row * x.stride + (uint32_t)u.h * kHeadBytes + 16 * (l >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const v8*>(src + 64 * i);
    };
    auto lse_load = [&](const Unit& u) __attribute__((always_inline)) -> float2 {
        const int32_t row = min(max(u.w, 0) * 16 + (anew(lane) & 15), n - 1);
        return *reinterpret_cast<const float2*>(p.lse + ((int64_t)row * H + u.h) * 2);
    };
    v8 o1[4], o2[4];
    float2 lse = make_float2(0.f, 0.f);

    Places at = places(L.x1, lane);
    const uint32_t records = (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(uint32_t)(uintptr_t)(LdsPtr)&L.rec[0]);
    const u2* __restrict__ recs = reinterpret_cast<const u2*>(p.columns);
    // Two records of 32 references and 32 masks, two words per lane (the lists end in
    // four spare records, so a block is read whole).  They go to slots `to` and
    // `to` + 1 of four, `to` 0 or 2.
    auto fetch = [&](int32_t c) __attribute__((always_inline)) -> u2 {
        return recs[(int64_t)c * 32 + anew(lane)];
    };
    auto hand_out = [&](int32_t to, uint32_t h, u2 blk) __attribute__((always_inline)) {
        const int l = anew(lane);
        DiffRecord& rec = L.rec[to + (l >> 5)];
        const int pos = 2 * (l & 15);
        if (l & 16) {
            *reinterpret_cast<u2*>(&rec.rm[pos]) = blk;
        } else {
            u2 a, b, s;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool none = blk[i] >= p.no_ref;
                const uint32_t node =
                    (uint32_t)(((uint64_t)(blk[i] >> p.ref_shift) * p.ref_magic) >> 31);
                if constexpr (WIDE) {
                    a[i] = none ? kNoIdx : node;
                } else {
                    a[i] = none ? kNoRow : node * (uint32_t)p.x1.stride;
                    b[i] = none ? kNoRow : node * (uint32_t)p.x2.stride;
                }
                s[i] = none ? kNoRow : (node * H + h) * 16u;
            }
            *reinterpret_cast<u2*>(&rec.at1[pos]) = a;
            if constexpr (!WIDE) *reinterpret_cast<u2*>(&rec.at2[pos]) = b;
            if constexpr (PASS == kDiffColumns) *reinterpret_cast<u2*>(&rec.st[pos]) = s;
        }
    };

    v8 a[8], b[8];
    f2 stat = {0.f, 0.f};   // (columns) half of slot lane / 2's
    // the rows of the record in slot `rec`: 16 lanes each, four at a time
    auto load1 = [&](int32_t slot, uint32_t h) __attribute__((always_inline)) {
        // (the forward pass has the registers)
        const int l = PASS == kDiffForward ? lane : anew(lane), g = l >> 4, r = l & 15;
        const uint32_t extra = h * kHeadBytes + 16 * r;
        const DiffRecord& rec = L.rec[slot];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = diff_load<T, WIDE>(r1, p.x1, rec.at1[4 * i + g], extra);
    };
    auto load2 = [&](int32_t slot, uint32_t h) __attribute__((always_inline)) {
        // (the forward pass has the registers)
        const int l = PASS == kDiffForward ? lane : anew(lane), g = l >> 4, r = l & 15;
        const uint32_t extra = h * kHeadBytes + 16 * r;
        const DiffRecord& rec = L.rec[slot];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            b[i] = diff_load<T, WIDE>(r2, p.x2, WIDE ? rec.at1[4 * i + g] : rec.at2[4 * i + g], extra);
        if constexpr (PASS == kDiffColumns) {
            const int l = anew(lane);
            stat = __builtin_bit_cast(
                f2, __builtin_amdgcn_raw_buffer_load_b64(rst, rec.st[l >> 1] + 8 * (l & 1), 0, 0));
        }
    };

    DiffState st;
    Unit u, next;
    uint32_t tick = 0;
    uint64_t flagged = 0;     // (repair) units [base, base + 64) that are left
    uint32_t base = 0;
    if constexpr (MODE == kDiffMain) {
        if (p.queue) {
            tick = ticket();
            const uint32_t second = ticket();
            u = redeem(tick);
            tick = second;
        } else {
            u = of_share(blockIdx.x / kXcds * kDiffWaves + wave);
        }
    } else if constexpr (MODE == kDiffTeam) {
        const uint32_t gb = (uint32_t)logical_block(p.xcd_contiguous);
        u = unit(gb / H * kDiffWaves + wave, gb % H, true);
    } else {
        base = (blockIdx.x * kDiffWaves + wave) * kWave;
        u = unit(0, 0, false);
    }
    next = u;
    next.ce = next.cb;
    bool warm = false;        // u's own rows, first chunk and first records are on their way
    u2 blk = {0u, 0u};
    int32_t slot = 0;         // of the current chunk's record
    for (;;) {
        if constexpr (MODE == kDiffMain) {
            if (u.end) break;
            next = redeem(tick);
            if (!next.end) tick = ticket();
        } else if constexpr (MODE == kDiffRepair) {
            const uint32_t units = (uint32_t)p.num_items * H;
            while (!flagged) {
                if (base >= units) return;
                flagged = __ballot(base + lane < units && p.odd[min(base + lane, units - 1)] != 0u);
                if (!flagged) base += gridDim.x * kDiffWaves * kWave;
            }
            const uint32_t at = base + __builtin_ctzll(flagged);
            flagged &= flagged - 1;
            if (!flagged) base += gridDim.x * kDiffWaves * kWave;
            u = unit(at / H, at % H, true);
        }
        [[maybe_unused]] uint64_t odd_sums = 0;   // bit 4 t + v: acc[t][v] has an odd value on an edge
        int sweep = MODE == kDiffRepair ? kSweepMark : kSweepPlain;
        while (u.w >= 0) {
            clear(st);
            if (PASS != kDiffForward && !Half<T>::kRange) st.x[0] = st.x[1] = 0.f;
            if (!warm) {
                own_load(p.own1, u, o1);
                if constexpr (PASS != kDiffForward) own_load(p.own2, u, o2);
                if constexpr (PASS == kDiffRows) lse = lse_load(u);
                slot = 0;
                if (u.cb < u.ce) {
                    blk = fetch(u.cb);
                    wave_lds_order();
                    hand_out(0, u.h, blk);
                    wave_lds_order();
                    load1(0, u.h);
                    load2(0, u.h);
                }
            }
            // the block of records after u's first, or the next unit's first
            const bool go_on = MODE == kDiffMain && next.cb < next.ce;
            auto fetch_after = [&](int32_t c) __attribute__((always_inline)) -> u2 {
                return c + kBlockRecs < u.ce ? fetch(c + kBlockRecs) : fetch(go_on ? next.cb : u.cb);
            };
            if (u.cb < u.ce) blk = fetch_after(u.cb);
            // |p_1 - lam p_2| <= 1 + |lam|: binary16's range needs lam out of it, and kLift
            float fit = 1.f, fit_lam = u.lam;   // (uniform)
            if constexpr (PASS == kDiffColumns && Half<T>::kRange) {
                fit = uniform(kLift<T> / __builtin_fmaxf(1.f, __builtin_fabsf(u.lam)));
                fit_lam = uniform(fit * u.lam);
            }
            if constexpr (PASS == kDiffRows) {
                const int l = anew(lane);
                const int32_t row = u.w * 16 + l;
                // (the columns' pass finds them beside D)
                if (l < 16 && row < n && (MODE != kDiffTeam || wave == 0))
                    *reinterpret_cast<float2*>(p.stats + ((int64_t)row * H + u.h) * 4) = lse;
                lse.x -= kLiftLog2<T>;
                lse.y -= kLiftLog2<T>;
                // The matrix cores' sums are rounded towards one side, by some 2^-30 of
                // g: nothing, but for dlam, where it adds up over all rows (500,000 of
                // them: 1.4e-5 of it).  Odd rows take -do, and their sums of p g are
                // negated at the end, so that it cancels.
                const uint32_t flip = (r & 1) ? 0x80008000u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o2[i] = __builtin_bit_cast(v8, __builtin_bit_cast(u4, o2[i]) ^ flip);
            }
            if constexpr (PASS == kDiffForward) {
                // (the running maxima are of s c with c > 0)
                const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o1[i] = __builtin_bit_cast(v8, __builtin_bit_cast(u4, o1[i]) ^ flip);
            }
            for (int32_t c = u.cb; c < u.ce; ++c) {
                const bool last = c + 1 == u.ce;
                if (((c - u.cb) % kBlockRecs) == 0) {
                    // the block ahead, so that the next chunk's record is there
                    const bool own_block = c + kBlockRecs < u.ce;
                    hand_out((slot & 2) ^ 2, own_block ? u.h : next.h, blk);
                    if (own_block) blk = fetch_after(c + kBlockRecs);
                }
                const uint32_t masks = records + slot * (uint32_t)sizeof(DiffRecord) +
                                       (uint32_t)offsetof(DiffRecord, rm);
                // where the stream goes on: the unit's next chunk, or the next unit's first
                const int32_t ahead = last ? (slot & 2) ^ 2 : (slot + 1) & 3;
                const uint32_t ahead_h = last ? (uint32_t)next.h : (uint32_t)u.h;
                const bool more = !last || go_on;
                held(at);
                write_rows(at, 0, a);
                wave_lds_order();
                if (more) load1(ahead, ahead_h);
                // S^T of both maps: slots 4g.. and 16 + 4g.. of row r
                f4 s[2][2];
                if constexpr (PASS != kDiffRows) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            s[m][t] = products<T, 2>(at, kHalfStage * t, 2 * m, o1);
                }
                write_rows(at, kStageBytes, b);
                if constexpr (PASS == kDiffColumns) {
                    *reinterpret_cast<f2*>(&L.stats[2 * anew(lane)]) = stat;
                }
                wave_lds_order();
                // (columns in binary16, with range_update's registers: only once the
                // weights are made)
                constexpr bool kLate = PASS == kDiffColumns && Half<T>::kRange;
                if (!kLate && more) load2(ahead, ahead_h);
                if (PASS == kDiffForward && last && go_on) own_load(p.own1, next, o1);
                if constexpr (PASS == kDiffForward) {
                    Attends on;
                    attends(masks, lane, on);
                    float pw[2][8];
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        map_update(st, m, s[m][0], s[m][1], on, p.scale_log2, pw[m]);
                    if (MODE != kDiffMain && sweep != kSweepPlain) {
                        if (sweep == kSweepMark) edge_weights(pw, on);
                        replace_odd<T>(at, kStageBytes, kStageBytes, sweep);
                    }
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const Tiles<T> x(at, kStageBytes, 4 * v);
#pragma unroll
                        for (int m = 0; m < 2; ++m) x.mix(pw[m], &st.acc[8 * m + 4 * v]);
                    }
                } else {
                    // g = do . v for the same pairs
                    f4 gs[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        gs[t] = products<T, 4>(at, kStageBytes + kHalfStage * t, 0, o2);
                    if (PASS == kDiffRows && last && go_on) own_load(p.own2, next, o2);
                    if constexpr (PASS == kDiffRows) {
                        // (a map's logits where its weights are made: registers)
                        const bool replaced = MODE != kDiffMain && sweep != kSweepPlain;
                        if (replaced) replace_odd<T>(at, 0, kStageBytes, sweep);
                        const uint32_t mixed = replaced ? kStageBytes : 0;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            f4 sm[2];
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                sm[t] = products<T, 2>(at, kHalfStage * t, 2 * m, o1);
                            if (m == 1 && last && go_on) own_load(p.own1, next, o1);
                            Attends on;
                            attends(masks, lane, on);
                            float pw[1][8], pg[1][8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float e = fast_exp2(lifted<T>(
                                    __builtin_fmaf(sm[j >> 2][j & 3], p.scale_log2,
                                                   m ? -lse.y : -lse.x),
                                    kLiftLog2<T> + 1.f));
                                pw[0][j] = where(on[j], e);
                                st.z[m] += pw[0][j];
                            }
                            if (MODE != kDiffMain && sweep == kSweepMark) edge_weights(pw, on);
                            const Tiles<T> x(at, mixed, 4 * m);
                            x.mix(pw[0], &st.acc[8 + 4 * m]);
                            __builtin_amdgcn_sched_barrier(0);
                            attends(masks, lane, on);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                pg[0][j] = where(on[j], pw[0][j] * gs[j >> 2][j & 3]);
                                st.y[m] += pg[0][j];
                            }
                            if (MODE != kDiffMain && sweep == kSweepMark) edge_weights(pg, on);
                            range_update<T>(st, m, pg[0]);
                            x.mix(pg[0], &st.acc[4 * m]);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        if (last && go_on) lse = lse_load(next);
                    } else {
                        Attends on;
                        if (MODE != kDiffMain && sweep != kSweepPlain) {
                            replace_odd<T>(at, 0, 0, sweep);
                            replace_odd<T>(at, kStageBytes, kStageBytes, sweep);
                        }
                        float pw[2][8];
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            __builtin_amdgcn_sched_barrier(0);
                            attends(masks, lane, on);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                pw[m][j] = where(
                                    on[j], fast_exp2(lifted<T>(
                                               __builtin_fmaf(s[m][j >> 2][j & 3], p.scale_log2,
                                                              -L.stats[4 * slot_of(g, j) + m]),
                                               0.f)));
                        }
                        __builtin_amdgcn_sched_barrier(0);
                        if (kLate && more) load2(ahead, ahead_h);
                        {
                            float wv[1][8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) wv[0][j] = pw[0][j] * fit - pw[1][j] * fit_lam;
                            if (MODE != kDiffMain && sweep == kSweepMark) edge_weights(wv, on);
#pragma unroll
                            for (int v = 0; v < 2; ++v) {
                                Tiles<T>(at, kStageBytes, 4 * v).mix(wv[0], &st.acc[8 + 4 * v]);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            attends(masks, lane, on);
                            float ds[1][8];
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                ds[0][j] = where(on[j], pw[m][j] * (gs[j >> 2][j & 3] -
                                                                    L.stats[4 * slot_of(g, j) + 2 + m]));
                            if (MODE != kDiffMain && sweep == kSweepMark) edge_weights(ds, on);
                            __builtin_amdgcn_sched_barrier(0);
                            range_update<T>(st, m, ds[0]);
                            v8 hi, lo;
                            split8<T>(ds[0], hi, lo);
                            // (two tiles at a time: registers)
#pragma unroll
                            for (int v = 0; v < 2; ++v) {
                                __builtin_amdgcn_sched_barrier(0);
                                Tiles<T, 2>(at, 0, 4 * m + 2 * v).mix(hi, lo, &st.acc[4 * m + 2 * v]);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
                wave_lds_order();
                slot = ahead;
            }
            warm = u.cb < u.ce && go_on;
            if (PASS == kDiffColumns && warm) {   // (inside the loop they cost it registers)
                own_load(p.own1, next, o1);
                own_load(p.own2, next, o2);
            }
            if (sweep == kSweepPlain) {
                // (x - x is 0 for finite x, NaN otherwise)
                float odd = 0.f;
#pragma unroll
                for (int t = 0; t < 16; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v) odd += st.acc[t][v] - st.acc[t][v];
                const bool any = __ballot(odd != 0.f) != 0;
                if constexpr (MODE == kDiffMain) {
                    if (lane == 0) p.odd[u.item * H + u.h] = any;
                    break;
                }
                if (!any) break;
                sweep = kSweepMark;
            } else if (sweep == kSweepMark) {
#pragma unroll
                for (int t = 0; t < 16; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        odd_sums |= (uint64_t)(st.acc[t][v] != 0.f) << (4 * t + v);
                sweep = kSweepClean;
            } else {
#pragma unroll
                for (int t = 0; t < 16; ++t)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if ((odd_sums >> (4 * t + v)) & 1u) st.acc[t][v] = NAN;
                break;
            }
        }
        if (u.w < 0) {
            warm = false;
            if (MODE == kDiffMain && u.there && lane == 0) p.odd[u.item * H + u.h] = 0u;
        }
        if constexpr (MODE == kDiffTeam) break;
        if (u.w >= 0) {
            if (u.slot >= 0)   // a segment: its sums wait for diff_merge_kernel
                publish(st, p.partials + ((int64_t)u.slot * H + u.h) * kDiffPartial, lane);
            else
                diff_finish<T, PASS>(p, st, L.x1, u.w, u.h, u.lam, lane);
        }
        if constexpr (MODE == kDiffMain) u = next;
    }
    if constexpr (MODE == kDiffTeam) {
        // waves 2, 3 into 0, 1, then 1 into 0: two states fit the team's memory
        // (a team's four are there or not together; teams have no segments)
        if (u.w < 0) return;
        float* area = reinterpret_cast<float*>(&lds_all[wave & 1]);
        __syncthreads();
        if (wave >= 2) publish(st, area, lane);
        __syncthreads();
        if (wave < 2) absorb<PASS>(st, area, lane);
        __syncthreads();
        if (wave == 1) publish(st, area, lane);
        __syncthreads();
        if (wave != 0) return;
        absorb<PASS>(st, reinterpret_cast<const float*>(&lds_all[1]), lane);
        diff_finish<T, PASS>(p, st, L.x1, u.w, u.h, u.lam, lane);
    }
}

__global__ void __launch_bounds__(256) clear_queues(uint32_t* __restrict__ queues, int32_t words)
{
    for (int32_t i = threadIdx.x; i < words; i += 256) queues[i] = 0u;
}

// The segments of a split window, in their order.
template <typename T, int PASS>
__global__ void __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(2)))
diff_merge_kernel(const DiffParams p)
{
    __shared__ __align__(16) _Float16 stage[16 * kRowHalves];
    const int lane = threadIdx.x;
    const SplitInfo si = p.splits[blockIdx.x / (uint32_t)p.H];
    const int h = (int)(blockIdx.x % (uint32_t)p.H);
    DiffState st;
    clear(st);
    for (int32_t k = 0; k < si.nseg; ++k)
        absorb<PASS>(st, p.partials + ((int64_t)(si.first_slot + k) * p.H + h) * kDiffPartial, lane);
    diff_finish<T, PASS>(p, st, stage, si.w, h, p.lam[h], lane);
}

// dlam[h] = -sum of its windows' shares, in one fixed order.
__global__ void __launch_bounds__(1024)
diff_dlam_kernel(const float* __restrict__ parts, int32_t W, float* __restrict__ dlam)
{
    __shared__ double lds[1024 / kWave];
    const float* src = parts + (int64_t)blockIdx.x * W;
    double s = 0.0;
    for (int32_t i = threadIdx.x; i < W; i += 32 * 1024) {
        float x[32];   // (in one batch: the loads' latency is all there is)
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = src[min(i + k * 1024, W - 1)];
#pragma unroll
        for (int k = 0; k < 32; ++k) s += i + k * 1024 < W ? x[k] : 0.f;
    }
    s = wave_sum(s);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 1024 / kWave; ++i) t += lds[i];
        dlam[blockIdx.x] = (float)-t;
    }
}

__global__ void warm_diff_kernel() {}

hipError_t warm_diff(hipStream_t s)
{
    hipLaunchKernelGGL(warm_diff_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

constexpr int64_t kDiffResident = 512;   // workgroups: two per CU, by their LDS
constexpr int32_t kRepairGroups = 256;

// Four-unit workgroups of each XCD's share of a plan's items.
static int64_t share_groups(const f3s_plan* plan)
{
    return ceil_div(ceil_div(plan->masked.num_items, kXcds) * plan->H, kDiffWaves);
}
// With a queue: two units for each wave and more.  (Below that it would be a launch
// more for nothing ahead to load.)
static bool has_queue(const f3s_plan* plan)
{
    return plan->masked.team == 1 && kXcds * share_groups(plan) >= 2 * kDiffResident;
}

template <typename T, int PASS, bool WIDE>
static void launch_diff(const DiffParams& p, const f3s_plan* plan, hipStream_t st)
{
    if (plan->masked.team > 1) {
        hipLaunchKernelGGL((diff_kernel<T, PASS, WIDE, kDiffTeam>),
                           dim3((unsigned)(p.num_items / kTeamSmall * p.H)),
                           dim3(kTeamSmall * kWave), 0, st, p);
        return;
    }
    const int64_t groups = has_queue(plan) ? kDiffResident : kXcds * share_groups(plan);
    hipLaunchKernelGGL((diff_kernel<T, PASS, WIDE, kDiffMain>), dim3((unsigned)groups),
                       dim3(kDiffWaves * kWave), 0, st, p);
    const int64_t units = p.num_items * p.H;
    hipLaunchKernelGGL((diff_kernel<T, PASS, WIDE, kDiffRepair>),
                       dim3((unsigned)std::min<int64_t>(kRepairGroups,
                                                        ceil_div(units, kDiffWaves * kWave))),
                       dim3(kDiffWaves * kWave), 0, st, p);
    if (p.num_split > 0)
        hipLaunchKernelGGL((diff_merge_kernel<T, PASS>), dim3((unsigned)(p.num_split * p.H)),
                           dim3(kWave), 0, st, p);
}

template <int PASS>
static f3s_status launch_pass(DiffParams p, const f3s_plan* plan, int32_t dtype, float scale,
                              hipStream_t st)
{
    const f3s_item_set& set = plan->masked;
    p.items = reinterpret_cast<const Item*>(set.items.ptr);
    p.num_items = set.num_items;
    p.splits = reinterpret_cast<const SplitInfo*>(set.splits.ptr);
    p.num_split = set.num_split;
    p.chunk_base = reinterpret_cast<const int32_t*>(plan->chunk_base.ptr);
    p.columns = reinterpret_cast<const uint32_t*>(plan->columns.ptr);
    p.W = plan->W;
    p.H = plan->H;
    p.xcd_contiguous = plan->xcd_contiguous;
    const bool nodes = wide_features(p.n, p.H);
    p.ref_shift = nodes ? 0 : 7;
    p.ref_magic = nodes ? 1u << 31 : (uint32_t)ceil_div((int64_t)1 << 31, p.H);
    p.no_ref = nodes ? kNoIdx : kNoRow;
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
    // (forward: q is negated for a negative scale; 0 x -inf is no logit)
    if (PASS == kDiffForward) p.scale_log2 = std::max(std::fabs(p.scale_log2), FLT_MIN);
    if (p.num_items <= 0) return F3S_OK;
    F3S_REQUIRE(p.num_items * p.H < ((int64_t)1 << 31) && (set.team == 1 || set.team == kTeamSmall),
                "differential attention: too many work items");
    // Offsets of 32 bits where every streamed tensor ends below kNoRow.
    const int64_t head = (int64_t)p.H * kHeadBytes;
    auto end = [&](const DiffRows& x) { return (int64_t)(p.n - 1) * (int64_t)x.stride + head; };
    const bool wide = end(p.x1) > (int64_t)kNoRow || end(p.x2) > (int64_t)kNoRow;
    if (!wide) {
        p.x1.bytes = (uint32_t)end(p.x1);
        p.x2.bytes = (uint32_t)end(p.x2);
    }
    if (p.stats) {
        const int64_t bytes = (int64_t)p.n * p.H * 16;
        if (bytes > (int64_t)kNoRow) {
            set_error("differential attention: n * H of 2^28 and more has no gradient here");
            return F3S_EUNSUPPORTED;
        }
        p.stats_bytes = (uint32_t)bytes;
    }
    if (dtype == F3S_F16) {
        if (wide) launch_diff<_Float16, PASS, true>(p, plan, st);
        else launch_diff<_Float16, PASS, false>(p, plan, st);
    } else {
        if (wide) launch_diff<__bf16, PASS, true>(p, plan, st);
        else launch_diff<__bf16, PASS, false>(p, plan, st);
    }
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

static size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

static size_t partial_bytes(const f3s_plan* plan)
{
    return round_up(sizeof(float) * kDiffPartial * (size_t)plan->H *
                    (size_t)plan->masked.num_slots);
}

// Workspace of a pass: its queues (a call's passes' side by side at the start), the
// marks of its units, its segments' sums.
constexpr size_t kQueueBytes = sizeof(uint32_t) * kXcds * kQueueStride;
struct PassSpace {
    size_t odd, partials, bytes;
};
static PassSpace pass_space(const f3s_plan* plan)
{
    PassSpace s{0, 0, 0};   // (teams merge in LDS)
    if (plan->masked.team == 1) {
        s.odd = 2 * kQueueBytes;
        s.partials = s.odd + round_up(sizeof(uint32_t) * (size_t)plan->masked.num_items * plan->H);
        s.bytes = s.partials + partial_bytes(plan);
    }
    return s;
}
static void set_space(DiffParams& p, const f3s_plan* plan, char* ws, int pass)
{
    const PassSpace s = pass_space(plan);
    p.queue = has_queue(plan) ? reinterpret_cast<uint32_t*>(ws + pass * kQueueBytes) : nullptr;
    p.odd = reinterpret_cast<uint32_t*>(ws + s.odd);
    p.partials = reinterpret_cast<float*>(ws + s.partials);
}
static void launch_clear(const DiffParams& p, int passes, hipStream_t st)
{
    if (p.queue)
        hipLaunchKernelGGL(clear_queues, dim3(1), dim3(256), 0, st, p.queue,
                           passes * kXcds * kQueueStride);
}

static f3s_status check_plan(const f3s_plan* plan, int32_t n, int32_t H, const char* who)
{
    if (!plan || plan->compiled_n < 0 || plan->compiled_n != n || plan->H != H) {
        set_error(std::string(who) + ": needs a plan compiled for this n and H");
        return F3S_EINVAL;
    }
    return F3S_OK;
}

// Rows at 16-byte boundaries, wide enough for the heads.
static bool rows_ok(const void* ptr, int64_t stride, int32_t H)
{
    return ptr && ((uintptr_t)ptr & 15) == 0 && stride % 8 == 0 && stride >= (int64_t)H * kHeadD &&
           stride < ((int64_t)1 << 30);
}

static DiffRows rows_of(const void* ptr, int64_t stride)
{
    return DiffRows{static_cast<const char*>(ptr), (uint64_t)stride * 2, 0};
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_diff_attention_workspace(const f3s_plan* plan, const f3s_plan* reversed,
                                        int64_t* bytes)
{
    F3S_REQUIRE(plan && bytes, "f3s_diff_attention_workspace: NULL pointer");
    size_t need = pass_space(plan).bytes;
    if (reversed) {
        const size_t cells = (size_t)std::max(plan->compiled_n, 0) * plan->H;
        need = std::max(need, pass_space(reversed).bytes) + round_up(cells * 16) +
               round_up(sizeof(float) * (size_t)plan->W * plan->H);
    }
    *bytes = (int64_t)need;
    return F3S_OK;
}

f3s_status f3s_diff_attention_fwd(const f3s_plan* plan, const uint16_t* Q, int64_t q_stride,
                                  const uint16_t* K, int64_t k_stride, const uint16_t* V,
                                  int64_t v_stride, const float* lam, uint16_t* O, int64_t o_stride,
                                  float* lse, int32_t dtype, int32_t n, int32_t H, float scale,
                                  void* workspace, int64_t workspace_bytes, void* stream)
{
    F3S_REQUIRE(n >= 0, "f3s_diff_attention_fwd: negative n");
    F3S_REQUIRE(dtype == F3S_F16 || dtype == F3S_BF16, "f3s_diff_attention_fwd: unknown dtype");
    F3S_TRY(check_plan(plan, n, H, "f3s_diff_attention_fwd"));
    if (n == 0) return F3S_OK;
    F3S_REQUIRE(rows_ok(Q, q_stride, H) && rows_ok(K, k_stride, H) && rows_ok(V, v_stride, H) &&
                    rows_ok(O, o_stride, H) && lam && ((uintptr_t)lse & 7) == 0,
                "f3s_diff_attention_fwd: NULL or misaligned pointer, or a row stride that is no "
                "multiple of 8 or below H * 128");
    F3S_REQUIRE(workspace_bytes >= (int64_t)pass_space(plan).bytes &&
                    (workspace || pass_space(plan).bytes == 0) && ((uintptr_t)workspace & 15) == 0,
                "f3s_diff_attention_fwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    DiffParams p{};
    p.x1 = rows_of(K, k_stride);
    p.x2 = rows_of(V, v_stride);
    p.own1 = rows_of(Q, q_stride);
    p.out1 = rows_of(O, o_stride);
    p.lam = lam;
    p.lse = lse;
    p.n = n;
    set_space(p, plan, static_cast<char*>(workspace), 0);
    launch_clear(p, 1, as_stream(stream));
    return launch_pass<kDiffForward>(p, plan, dtype, scale, as_stream(stream));
}

f3s_status f3s_diff_attention_bwd(const f3s_plan* plan, const f3s_plan* reversed,
                                  const uint16_t* Q, int64_t q_stride, const uint16_t* K,
                                  int64_t k_stride, const uint16_t* V, int64_t v_stride,
                                  const float* lam, const float* lse, const uint16_t* dO,
                                  int64_t do_stride, uint16_t* dQ, int64_t dq_stride, uint16_t* dK,
                                  int64_t dk_stride, uint16_t* dV, int64_t dv_stride, float* dlam,
                                  int32_t dtype, int32_t n, int32_t H, float scale, void* workspace,
                                  int64_t workspace_bytes, void* stream)
{
    F3S_REQUIRE(n >= 0, "f3s_diff_attention_bwd: negative n");
    F3S_REQUIRE(dtype == F3S_F16 || dtype == F3S_BF16, "f3s_diff_attention_bwd: unknown dtype");
    F3S_TRY(check_plan(plan, n, H, "f3s_diff_attention_bwd"));
    F3S_TRY(check_plan(reversed, n, H, "f3s_diff_attention_bwd (reversed)"));
    F3S_REQUIRE(lam && dlam, "f3s_diff_attention_bwd: NULL pointer");
    F3S_REQUIRE(n == 0 || (rows_ok(Q, q_stride, H) && rows_ok(K, k_stride, H) &&
                           rows_ok(V, v_stride, H) && rows_ok(dO, do_stride, H) &&
                           rows_ok(dQ, dq_stride, H) && rows_ok(dK, dk_stride, H) &&
                           rows_ok(dV, dv_stride, H) && lse && ((uintptr_t)lse & 7) == 0),
                "f3s_diff_attention_bwd: NULL or misaligned pointer, or a row stride that is no "
                "multiple of 8 or below H * 128");
    int64_t need = 0;
    F3S_TRY(f3s_diff_attention_workspace(plan, reversed, &need));
    F3S_REQUIRE(workspace_bytes >= need && (workspace || need == 0) &&
                    ((uintptr_t)workspace & 15) == 0,
                "f3s_diff_attention_bwd: workspace too small");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    DiffParams p{};
    p.lam = lam;
    p.n = n;
    if (n > 0) {
        char* ws = static_cast<char*>(workspace);
        p.stats = reinterpret_cast<float*>(ws);
        p.dlam_parts = reinterpret_cast<float*>(ws + round_up((size_t)n * H * 16));
        char* spaces = ws + round_up((size_t)n * H * 16) + round_up(sizeof(float) * (size_t)plan->W * H);
        p.lse = const_cast<float*>(lse);
        DiffParams rows = p;
        rows.x1 = rows_of(K, k_stride);
        rows.x2 = rows_of(V, v_stride);
        rows.own1 = rows_of(Q, q_stride);
        rows.own2 = rows_of(dO, do_stride);
        rows.out1 = rows_of(dQ, dq_stride);
        set_space(rows, plan, spaces, 0);
        DiffParams cols = p;
        set_space(cols, reversed, spaces, 1);
        if (rows.queue) launch_clear(rows, 2, st);
        else launch_clear(cols, 1, st);
        F3S_TRY(launch_pass<kDiffRows>(rows, plan, dtype, scale, st));
        cols.x1 = rows_of(Q, q_stride);
        cols.x2 = rows_of(dO, do_stride);
        cols.own1 = rows_of(K, k_stride);
        cols.own2 = rows_of(V, v_stride);
        cols.out1 = rows_of(dK, dk_stride);
        cols.out2 = rows_of(dV, dv_stride);
        F3S_TRY(launch_pass<kDiffColumns>(cols, reversed, dtype, scale, st));
    }
    hipLaunchKernelGGL(diff_dlam_kernel, dim3((unsigned)H), dim3(1024), 0, st, p.dlam_parts,
                       n > 0 ? plan->W : 0, dlam);
    F3S_HIP(hipGetLastError());
    return F3S_OK;
}

}  // extern "C"
