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
// their difference.  Sums and softmax statistics are in float32.
//
// A value that is infinite or NaN reaches, through the matrix cores, rows of its
// window that have no edge to it (0 x inf).  So a window whose sums are not
// finite at the end is done twice more: once to mark the sums that have such a
// value on an edge of theirs, which become NaN, and once without those values.
#include <algorithm>

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
    int32_t refs_are_nodes; // column lists of node indices, else of node * H * 128
    uint32_t heads_magic;   // ceil(2^31 / H): (x * magic) >> 31 = x / H for x < 2^25
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
        const f4 a = *reinterpret_cast<const f4*>(&src[(t * kWave + lane) * 4]);
        s.acc[t] += c < 2 ? a * theirs[c] : a;
    }
}

// One chunk's slots of a record: byte offsets into x1 and x2 (narrow) or node
// indices (wide), row masks, and byte offsets into stats.
struct DiffRecord {
    uint32_t at1[kChunk], at2[kChunk], rm[kChunk], st[kChunk];
};
constexpr int kBlockRecs = 2;   // records read, converted and handed out together
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

// acc[i][t] += sum over the chunk's slots of w[i] (the lane's slots of row r)
// times the 16 dims of tile t0 + t, four tiles.
template <typename T, int N>
__device__ __forceinline__ void mix(const Places& p, uint32_t stage, int t0,
                                    const typename Half<T>::v8 (&w)[N], f4* const (&acc)[N])
{
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const typename Half<T>::v8 x = transposed<T>(p, stage, t0 + t);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i][t] = Half<T>::mfma(x, w[i], acc[i][t]);
    }
}

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

// A staged chunk's values: MARK: 1 where infinite or NaN, else 0; CLEAN: 0 there.
enum Sweep : int { kSweepPlain = 0, kSweepMark = 1, kSweepClean = 2 };
template <typename T>
__device__ __forceinline__ void replace_odd(const Places& p, uint32_t stage, int sweep)
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
        lds_write(at, x);
    }
    wave_lds_order();
}

template <int N>
__device__ __forceinline__ void edge_weights(float (&w)[N][8], uint32_t valid)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = (valid >> j) & 1u ? 1.f : 0.f;
}

// Running maximum of one map (log2): moved when a chunk's exceeds it by more
// than kLazy.  p[j] = 2^(x - m), 0 where not attended; l is the lane's share.
__device__ __forceinline__ void map_update(DiffState& st, int c, const f4 s0, const f4 s1,
                                           uint32_t valid, float scale_log2, float (&p)[8])
{
    float x[8];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        x[v] = ((valid >> v) & 1u) ? s0[v] * scale_log2 : -INFINITY;
        x[4 + v] = ((valid >> (4 + v)) & 1u) ? s1[v] * scale_log2 : -INFINITY;
    }
    float cm = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) cm = __builtin_fmaxf(cm, x[j]);
    cm = row_max4(cm);
    if (__ballot(cm > st.x[c] + kLazy)) {
        if (cm > st.x[c] + kLazy) {
            const float corr = fast_exp2(st.x[c] - cm);
            st.y[c] *= corr;
            rescale<kDiffForward>(st, c, corr);
            st.x[c] = cm;
        }
    }
    const float mu = st.x[c] == -INFINITY ? 0.f : st.x[c];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        p[j] = fast_exp2(x[j] - mu);
        st.y[c] += p[j];
    }
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
                                            int32_t w, int h, int lane)
{
    const int g = lane >> 4, r = lane & 15;
    const int32_t row = w * 16 + r;
    const uint32_t head_off = (uint32_t)h * kHeadBytes;
    const float lam = p.lam[h];
    if constexpr (PASS == kDiffForward) {
        const float l1 = over_groups(st.y[0]), l2 = over_groups(st.y[1]);
        const bool some = l1 != 0.f;   // (a row of NaN is some)
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
        const float back = Half<T>::kRange ? __builtin_fmaxf(1.f, __builtin_fabsf(lam)) : 1.f;
        store_rows<T>(p.out1, stage, w, p.n, head_off, lane, [&](int t) {
            return t < 4 ? p.scale * (st.acc[t] * f1) : -lam * p.scale * (st.acc[t] * f2);
        });
        store_rows<T>(p.out2, stage, w, p.n, head_off, lane,
                      [&](int t) { return st.acc[8 + t] * back; });
    }
}

template <typename T, int PASS, bool WIDE, int WPG, bool TEAM>
__global__ void __launch_bounds__(kWave * WPG) __attribute__((amdgpu_waves_per_eu(2)))
diff_kernel(const DiffParams p)
{
    typedef typename Half<T>::v8 v8;
    static_assert(!TEAM || WPG == kTeamSmall, "a team fills its workgroup");
    __shared__ DiffLds lds_all[WPG];
    const int wave = threadIdx.x / kWave;
    const int lane = threadIdx.x % kWave;
    const int g = lane >> 4, r = lane & 15;
    DiffLds& L = lds_all[wave];
    const int H = p.H;

    // wave -> (item, head).  A scheduled plan's items are eight interleaved shares,
    // share x for XCD x, and the dispatcher deals workgroups to the XCDs in turn:
    // workgroup b takes items of share b % 8, the heads of an item adjacent.
    int64_t item_idx;
    int h;
    if constexpr (TEAM) {
        const uint32_t gb = (uint32_t)logical_block(p.xcd_contiguous);
        item_idx = (int64_t)(gb / (uint32_t)H) * WPG + wave;
        h = (int)(gb % (uint32_t)H);
    } else {
        const uint32_t b = (uint32_t)logical_block(p.xcd_contiguous);
        const uint32_t at = b / kXcds * WPG + wave;
        item_idx = (int64_t)(at / (uint32_t)H) * kXcds + b % kXcds;
        if (p.xcd_contiguous) item_idx = (int64_t)((b * WPG + wave) / (uint32_t)H);
        h = (int)((p.xcd_contiguous ? b * WPG + wave : at) % (uint32_t)H);
    }
    if (item_idx >= p.num_items) return;   // (a team's four are there or not together)
    const Item it = p.items[item_idx];
    const int32_t w = it.w;
    if (w < 0 || w >= p.W) return;
    const int32_t n = p.n;
    const uint32_t head_off = (uint32_t)h * kHeadBytes;
    const float lam = p.lam[h];

    const __amdgpu_buffer_rsrc_t r1 = make_rsrc(p.x1.ptr, p.x1.bytes);
    const __amdgpu_buffer_rsrc_t r2 = make_rsrc(p.x2.ptr, p.x2.bytes);
    const __amdgpu_buffer_rsrc_t rst = make_rsrc(p.stats, p.stats_bytes);

    // ---- the window's own rows, in operand order: dims 32 f + 8 g .. of row r ----
    const int32_t row = w * 16 + r;
    auto own_load = [&](const DiffRows& x, v8 (&f)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = v8{};
            if (row < n)
                f[i] = *reinterpret_cast<const v8*>(x.ptr + row * x.stride + head_off + 64 * i + 16 * g);
        }
    };
    v8 o1[4], o2[4];
    own_load(p.own1, o1);
    if constexpr (PASS != kDiffForward) own_load(p.own2, o2);
    if constexpr (PASS == kDiffRows) {
        // The matrix cores' sums are rounded towards one side, by some 2^-30 of g:
        // nothing, but for dlam, where it adds up over all rows (500,000 of them:
        // 1.4e-5 of it).  Odd rows take -do, and their sums of p g are negated at
        // the end, so that it cancels.
        if (r & 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o2[i] = -o2[i];
        }
    }
    float lse1 = 0.f, lse2 = 0.f;
    if constexpr (PASS == kDiffRows) {
        if (row < n) {
            const float2 l = *reinterpret_cast<const float2*>(p.lse + ((int64_t)row * H + h) * 2);
            lse1 = l.x;
            lse2 = l.y;
            // (the columns' pass finds them beside D)
            if (g == 0 && (!TEAM || wave == 0))
                *reinterpret_cast<float2*>(p.stats + ((int64_t)row * H + h) * 4) = l;
        }
    }

    const int64_t cb = p.chunk_base[item_idx], ce = p.chunk_base[item_idx + 1];
    const uint32_t extra = head_off + 16 * r;   // rows are read 16 lanes each, four at a time
    Places at = places(L.x1, lane);
    const int rbit = (r & 1) ? 16 + (r >> 1) : (r >> 1);
    const u4* __restrict__ recs = reinterpret_cast<const u4*>(p.columns);
    // Two records of 32 references and 32 masks: lane l < 32 holds words 4 l .. 4 l + 3
    // (the lists end in four spare records, so a block is read whole).
    auto fetch = [&](int64_t c) __attribute__((always_inline)) -> u4 {
        return c < ce && lane < 16 * kBlockRecs ? recs[c * 16 + lane] : u4{0u, 0u, 0u, 0u};
    };
    auto hand_out = [&](int64_t c, u4 blk) __attribute__((always_inline)) {
        if (lane < 16 * kBlockRecs) {
            DiffRecord& rec = L.rec[(c - cb + (lane >> 4)) % (2 * kBlockRecs)];
            const int at = 4 * (lane & 7);
            if (lane & 8) {
                *reinterpret_cast<u4*>(&rec.rm[at]) = blk;
            } else {
                u4 a, b, s;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t ref = blk[i];
                    const bool none = p.refs_are_nodes ? ref == kNoIdx : ref >= kNoRow;
                    const uint32_t node =
                        p.refs_are_nodes ? ref
                                         : (uint32_t)(((uint64_t)(ref >> 7) * p.heads_magic) >> 31);
                    if constexpr (WIDE) {
                        a[i] = none ? kNoIdx : node;
                    } else {
                        a[i] = none ? kNoRow : node * (uint32_t)p.x1.stride;
                        b[i] = none ? kNoRow : node * (uint32_t)p.x2.stride;
                    }
                    s[i] = none ? kNoRow : (node * H + h) * 16u;
                }
                *reinterpret_cast<u4*>(&rec.at1[at]) = a;
                if constexpr (!WIDE) *reinterpret_cast<u4*>(&rec.at2[at]) = b;
                if constexpr (PASS == kDiffColumns) *reinterpret_cast<u4*>(&rec.st[at]) = s;
            }
        }
    };

    DiffState st;
    uint64_t odd_sums = 0;   // bit 4 t + v: acc[t][v] has an odd value on an edge
    int sweep = kSweepPlain;
    for (;;) {
        clear(st);
        if (PASS != kDiffForward && !Half<T>::kRange) st.x[0] = st.x[1] = 0.f;

        v8 a[8], b[8];
        f4 stat = {0.f, 0.f, 0.f, 0.f};
        u4 blk = fetch(cb);
        wave_lds_order();
        hand_out(cb, blk);
        wave_lds_order();
        blk = fetch(cb + kBlockRecs);
        auto load1 = [&](int64_t c) __attribute__((always_inline)) {
            const DiffRecord& rec = L.rec[(c - cb) % (2 * kBlockRecs)];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                a[i] = diff_load<T, WIDE>(r1, p.x1, rec.at1[4 * i + g], extra);
        };
        auto load2 = [&](int64_t c) __attribute__((always_inline)) {
            const DiffRecord& rec = L.rec[(c - cb) % (2 * kBlockRecs)];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                b[i] = diff_load<T, WIDE>(r2, p.x2, WIDE ? rec.at1[4 * i + g] : rec.at2[4 * i + g],
                                          extra);
            if constexpr (PASS == kDiffColumns) {
                const uint32_t at = lane < kChunk ? rec.st[lane] : kNoRow;
                stat = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rst, at, 0, 0));
            }
        };
        if (cb < ce) {
            load1(cb);
            load2(cb);
        }
        for (int64_t c = cb; c < ce; ++c) {
            if ((c - cb) % kBlockRecs == 0) {
                // the next block's records, so that the next chunk's are there
                hand_out(c + kBlockRecs, blk);
                blk = fetch(c + 2 * kBlockRecs);
            }
            const DiffRecord& rec = L.rec[(c - cb) % (2 * kBlockRecs)];
            const uint4 ra = *reinterpret_cast<const uint4*>(&rec.rm[4 * g]);
            const uint4 rb = *reinterpret_cast<const uint4*>(&rec.rm[16 + 4 * g]);
            const uint32_t valid =
                ((ra.x >> rbit) & 1u) | (((ra.y >> rbit) & 1u) << 1) |
                (((ra.z >> rbit) & 1u) << 2) | (((ra.w >> rbit) & 1u) << 3) |
                (((rb.x >> rbit) & 1u) << 4) | (((rb.y >> rbit) & 1u) << 5) |
                (((rb.z >> rbit) & 1u) << 6) | (((rb.w >> rbit) & 1u) << 7);
            held(at);
            write_rows(at, 0, a);
            wave_lds_order();
            if (c + 1 < ce) load1(c + 1);
            // S^T of both maps: slots 4g.. and 16 + 4g.. of row r
            f4 s[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    s[m][t] = products<T, 2>(at, kHalfStage * t, 2 * m, o1);
            write_rows(at, kStageBytes, b);
            if constexpr (PASS == kDiffColumns) {
                if (lane < kChunk) *reinterpret_cast<f4*>(&L.stats[4 * lane]) = stat;
            }
            wave_lds_order();
            if (c + 1 < ce) load2(c + 1);
            if constexpr (PASS == kDiffForward) {
                float pw[2][8];
#pragma unroll
                for (int m = 0; m < 2; ++m)
                    map_update(st, m, s[m][0], s[m][1], valid, p.scale_log2, pw[m]);
                if (sweep != kSweepPlain) {
                    if (sweep == kSweepMark) edge_weights(pw, valid);
                    replace_odd<T>(at, kStageBytes, sweep);
                }
                v8 wh[4];
                split8<T>(pw[0], wh[0], wh[1]);
                split8<T>(pw[1], wh[2], wh[3]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    f4* const to[4] = {&st.acc[4 * u], &st.acc[4 * u], &st.acc[8 + 4 * u],
                                       &st.acc[8 + 4 * u]};
                    mix<T>(at, kStageBytes, 4 * u, wh, to);
                }
            } else {
                // g = do . v for the same pairs
                f4 gs[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    gs[t] = products<T, 4>(at, kStageBytes + kHalfStage * t, 0, o2);
                if constexpr (PASS == kDiffRows) {
                    if (sweep != kSweepPlain) replace_odd<T>(at, 0, sweep);
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        float pw[1][8], pg[1][8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const bool on = (valid >> j) & 1u;
                            const float x = fast_exp2(__builtin_fmaf(s[m][j >> 2][j & 3],
                                                                     p.scale_log2,
                                                                     m ? -lse2 : -lse1));
                            pw[0][j] = on ? x : 0.f;
                            pg[0][j] = on ? x * gs[j >> 2][j & 3] : 0.f;
                            st.y[m] += pg[0][j];
                            st.z[m] += pw[0][j];
                        }
                        if (sweep == kSweepMark) {
                            edge_weights(pg, valid);
                            edge_weights(pw, valid);
                        }
                        range_update<T>(st, m, pg[0]);
                        v8 wh[4];
                        split8<T>(pg[0], wh[0], wh[1]);
                        split8<T>(pw[0], wh[2], wh[3]);
                        f4* const to[4] = {&st.acc[4 * m], &st.acc[4 * m], &st.acc[8 + 4 * m],
                                           &st.acc[8 + 4 * m]};
                        mix<T>(at, 0, 4 * m, wh, to);
                    }
                } else {
                    // |p_1 - lam p_2| <= 1 + |lam|: binary16's range needs lam out of it
                    const float fit =
                        Half<T>::kRange ? 1.f / __builtin_fmaxf(1.f, __builtin_fabsf(lam)) : 1.f;
                    float ds[2][8], wv[1][8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool on = (valid >> j) & 1u;
                        const float gj = gs[j >> 2][j & 3];
                        const f4 sj = *reinterpret_cast<const f4*>(&L.stats[4 * slot_of(g, j)]);
                        const float p1 =
                            fast_exp2(__builtin_fmaf(s[0][j >> 2][j & 3], p.scale_log2, -sj[0]));
                        const float p2 =
                            fast_exp2(__builtin_fmaf(s[1][j >> 2][j & 3], p.scale_log2, -sj[1]));
                        ds[0][j] = on ? p1 * (gj - sj[2]) : 0.f;
                        ds[1][j] = on ? p2 * (gj - sj[3]) : 0.f;
                        wv[0][j] = on ? p1 * fit - p2 * (lam * fit) : 0.f;
                    }
                    if (sweep != kSweepPlain) {
                        if (sweep == kSweepMark) {
                            edge_weights(ds, valid);
                            edge_weights(wv, valid);
                        }
                        replace_odd<T>(at, 0, sweep);
                        replace_odd<T>(at, kStageBytes, sweep);
                    }
                    v8 wh[2];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        range_update<T>(st, m, ds[m]);
                        split8<T>(ds[m], wh[0], wh[1]);
                        f4* const to[2] = {&st.acc[4 * m], &st.acc[4 * m]};
                        mix<T>(at, 0, 4 * m, wh, to);
                    }
                    split8<T>(wv[0], wh[0], wh[1]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f4* const to[2] = {&st.acc[8 + 4 * u], &st.acc[8 + 4 * u]};
                        mix<T>(at, kStageBytes, 4 * u, wh, to);
                    }
                }
            }
            wave_lds_order();
        }
        if (sweep == kSweepPlain) {
            // (x - x is 0 for finite x, NaN otherwise)
            float odd = 0.f;
#pragma unroll
            for (int t = 0; t < 16; ++t)
#pragma unroll
                for (int v = 0; v < 4; ++v) odd += st.acc[t][v] - st.acc[t][v];
            if (!__ballot(odd != 0.f)) break;
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

    if constexpr (TEAM) {
        // waves 2, 3 into 0, 1, then 1 into 0: two states fit the team's memory
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
    }
    if (it.slot >= 0) {   // a segment: its sums wait for diff_merge_kernel
        publish(st, p.partials + ((int64_t)it.slot * H + h) * kDiffPartial, lane);
        return;
    }
    diff_finish<T, PASS>(p, st, L.x1, w, h, lane);
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
    diff_finish<T, PASS>(p, st, stage, si.w, h, lane);
}

// dlam[h] = -sum of its windows' shares, in one fixed order.
__global__ void __launch_bounds__(1024)
diff_dlam_kernel(const float* __restrict__ parts, int32_t W, float* __restrict__ dlam)
{
    __shared__ double lds[1024 / kWave];
    double s = 0.0;
    const float* src = parts + (int64_t)blockIdx.x * W;
    for (int32_t i = threadIdx.x; i < W; i += 1024) s += src[i];
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

template <typename T, int PASS, bool WIDE>
static void launch_diff(const DiffParams& p, int32_t team, hipStream_t st)
{
    const int64_t waves = p.num_items * p.H;
    if (team > 1)
        hipLaunchKernelGGL((diff_kernel<T, PASS, WIDE, kTeamSmall, true>),
                           dim3((unsigned)(waves / kTeamSmall)), dim3(kTeamSmall * kWave), 0, st, p);
    else
        hipLaunchKernelGGL((diff_kernel<T, PASS, WIDE, 4, false>),
                           dim3((unsigned)(kXcds * ceil_div(ceil_div(p.num_items, kXcds) * p.H, 4))),
                           dim3(4 * kWave), 0, st, p);
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
    p.refs_are_nodes = wide_features(p.n, p.H);
    p.heads_magic = (uint32_t)ceil_div((int64_t)1 << 31, p.H);
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
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
        if (wide) launch_diff<_Float16, PASS, true>(p, set.team, st);
        else launch_diff<_Float16, PASS, false>(p, set.team, st);
    } else {
        if (wide) launch_diff<__bf16, PASS, true>(p, set.team, st);
        else launch_diff<__bf16, PASS, false>(p, set.team, st);
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
    size_t need = partial_bytes(plan);
    if (reversed) {
        const size_t cells = (size_t)std::max(plan->compiled_n, 0) * plan->H;
        need = std::max(need, partial_bytes(reversed)) + round_up(cells * 16) +
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
    F3S_REQUIRE(workspace_bytes >= (int64_t)partial_bytes(plan) &&
                    (workspace || partial_bytes(plan) == 0) && ((uintptr_t)workspace & 15) == 0,
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
    p.partials = static_cast<float*>(workspace);
    p.n = n;
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
        p.partials = reinterpret_cast<float*>(ws + round_up((size_t)n * H * 16) +
                                              round_up(sizeof(float) * (size_t)plan->W * H));
        p.lse = const_cast<float*>(lse);
        DiffParams rows = p;
        rows.x1 = rows_of(K, k_stride);
        rows.x2 = rows_of(V, v_stride);
        rows.own1 = rows_of(Q, q_stride);
        rows.own2 = rows_of(dO, do_stride);
        rows.out1 = rows_of(dQ, dq_stride);
        F3S_TRY(launch_pass<kDiffRows>(rows, plan, dtype, scale, st));
        DiffParams cols = p;
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
