// bsf_util.hip -- window ordering and block-sparse statistics on the GPU.
#include <rocprim/device/device_radix_sort.hpp>

#include "f3s_common.hpp"
#include "f3s_device.hpp"

namespace f3s {

__global__ void window_counts(const int32_t* __restrict__ offs, int32_t W,
                              uint32_t* __restrict__ counts, int32_t* __restrict__ iota)
{
    const int32_t w = blockIdx.x * blockDim.x + threadIdx.x;
    if (w >= W) return;
    const int32_t c = offs[w + 1] - offs[w];
    counts[w] = c > 0 ? (uint32_t)c : 0u;
    iota[w] = w;
}

// The order of up to kRankMax windows in one launch: every workgroup loads all
// windows' keys (tile count descending, then index: unique) into LDS and
// places 64 windows at their ranks, four lanes per window each counting the
// smaller keys in a quarter of the list.  O(W^2), about 5 us at kRankMax; the
// radix sort's five launches cost more host time than that up to there (1,251
// windows, call to completion: 38 us sorted, 25 us ranked), and past it the
// square overtakes.
constexpr int32_t kRankMax = 4096;
constexpr uint32_t kRankTiles = (1u << 20) - 1;   // a count above (no valid form has one) ties
static_assert(kRankMax <= 1 << 12, "the index takes 12 bits of the key, the count 20");

__global__ void __launch_bounds__(256)
rank_windows(const int32_t* __restrict__ offs, int32_t W, int32_t* __restrict__ order)
{
    __shared__ __align__(16) uint32_t key[kRankMax];
    const int tid = threadIdx.x;
    const int32_t quarter = (W + 15) / 16 * 4;   // keys a lane looks at, a multiple of 4
    for (int32_t i = tid; i < 4 * quarter; i += 256) {
        uint32_t k = 0xffffffffu;   // past the list: above every key
        if (i < W) {
            const int32_t c = offs[i + 1] - offs[i];
            k = (kRankTiles - min((uint32_t)max(c, 0), kRankTiles)) << 12 | (uint32_t)i;
        }
        key[i] = k;
    }
    __syncthreads();
    const int32_t i = blockIdx.x * 64 + tid / 4;
    const uint32_t ki = key[min(i, W - 1)];
    const uint4* mine = reinterpret_cast<const uint4*>(&key[(tid & 3) * quarter]);
    int32_t rank = 0;
    for (int32_t j = 0; j < quarter / 4; ++j) {
        const uint4 k = mine[j];
        rank += (k.x < ki) + (k.y < ki) + (k.z < ki) + (k.w < ki);
    }
    rank += __shfl_xor(rank, 1, kWave);
    rank += __shfl_xor(rank, 2, kWave);
    if (i < W && (tid & 3) == 0) order[rank] = i;
}

__global__ void __launch_bounds__(256)
bsf_stats_kernel(const int32_t* __restrict__ block_col, const uint16_t* __restrict__ tile_mask,
                 int64_t T, int32_t n, unsigned long long* __restrict__ out)
{
    __shared__ unsigned long long lds[2][256 / kWave];
    unsigned long long occ = 0, bits = 0;
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < T; t += stride) {
        const int64_t left = (int64_t)n - (int64_t)block_col[t] * 16;
        const uint32_t valid = left >= 16 ? 0xffffu : (left <= 0 ? 0u : ((1u << left) - 1u));
        if (tile_mask) {
            const uint4* mp = reinterpret_cast<const uint4*>(tile_mask + t * 16);
            const uint4 a = mp[0], b = mp[1];
            const uint32_t o = a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w;
            occ += __popc((o | (o >> 16)) & valid);
            bits += __popc(a.x) + __popc(a.y) + __popc(a.z) + __popc(a.w) + __popc(b.x) +
                    __popc(b.y) + __popc(b.z) + __popc(b.w);
        } else {
            occ += __popc(valid);
        }
    }
    occ = wave_sum(occ);
    bits = wave_sum(bits);
    const int wid = threadIdx.x / kWave;
    if ((threadIdx.x % kWave) == 0) {
        lds[0][wid] = occ;
        lds[1][wid] = bits;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned long long a = 0, b = 0;
        for (int i = 0; i < 256 / kWave; ++i) {
            a += lds[0][i];
            b += lds[1][i];
        }
        atomicAdd(out, a);
        atomicAdd(out + 1, b);
    }
}

// The reversed edges of a CSR: entries per column, their scan (the new row
// pointer), then every entry to the next free place of its column.  The order
// within a row is that of the atomics and differs from run to run; the converter
// does not mind it, and its lists come out the same.  256 entries per workgroup:
// the rows they span are found once, each entry's among those.
__global__ void __launch_bounds__(256)
clear_counts(int32_t* __restrict__ a, int64_t count)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) a[i] = 0;
}

__global__ void __launch_bounds__(256)
column_counts(const int32_t* __restrict__ col_idx, int64_t nnz, int32_t n,
              int32_t* __restrict__ counts)
{
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= nnz) return;
    const int32_t c = col_idx[e];
    if ((uint32_t)c < (uint32_t)n) atomicAdd(&counts[c], 1);
}

// The last of rows [lo, hi] that starts at or before entry e.
__device__ __forceinline__ int32_t row_of(const int32_t* __restrict__ row_ptr, int32_t lo,
                                          int32_t hi, int64_t e)
{
    while (lo < hi) {
        const int32_t mid = lo + (hi - lo + 1) / 2;
        if (row_ptr[mid] <= e) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(256)
reverse_fill(const int32_t* __restrict__ row_ptr, const int32_t* __restrict__ col_idx, int64_t nnz,
             int32_t n, const int32_t* __restrict__ out_ptr, int32_t* __restrict__ used,
             int32_t* __restrict__ out_idx)
{
    __shared__ int32_t span[2];
    const int64_t e0 = (int64_t)blockIdx.x * 256, e = e0 + threadIdx.x;
    if (threadIdx.x < 2)
        span[threadIdx.x] = row_of(row_ptr, 0, n - 1, threadIdx.x ? min(e0 + 255, nnz - 1) : e0);
    __syncthreads();
    if (e >= nnz) return;
    const int32_t c = col_idx[e];
    if ((uint32_t)c >= (uint32_t)n) return;
    const int32_t row = row_of(row_ptr, span[0], max(span[0], span[1]), e);
    const int64_t at = (int64_t)out_ptr[c] + atomicAdd(&used[c], 1);
    if (at < nnz) out_idx[at] = row;
}

__global__ void warm_bsf_util_kernel() {}

hipError_t warm_bsf_util(hipStream_t s)
{
    hipLaunchKernelGGL(warm_bsf_util_kernel, dim3(1), dim3(64), 0, s);
    return hipGetLastError();
}

}  // namespace f3s

using namespace f3s;

extern "C" {

f3s_status f3s_window_order(const int32_t* d_window_offsets, int32_t W, int32_t* d_order,
                            void* stream)
{
    F3S_REQUIRE(W >= 0, "f3s_window_order: negative W");
    if (W == 0) return F3S_OK;
    F3S_REQUIRE(d_window_offsets && d_order, "f3s_window_order: NULL pointer");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    if (W <= kRankMax) {
        hipLaunchKernelGGL(rank_windows, dim3((unsigned)ceil_div(W, 64)), dim3(256), 0, st,
                           d_window_offsets, W, d_order);
        F3S_HIP(hipGetLastError());
        F3S_HIP(hipStreamSynchronize(st));
        return F3S_OK;
    }
    StreamBuffer keys_in(st), keys_out(st), vals_in(st), tmp(st);
    F3S_TRY(keys_in.reserve(sizeof(uint32_t) * (size_t)W));
    F3S_TRY(keys_out.reserve(sizeof(uint32_t) * (size_t)W));
    F3S_TRY(vals_in.reserve(sizeof(int32_t) * (size_t)W));
    auto* ki = reinterpret_cast<uint32_t*>(keys_in.ptr);
    auto* ko = reinterpret_cast<uint32_t*>(keys_out.ptr);
    auto* vi = reinterpret_cast<int32_t*>(vals_in.ptr);
    hipLaunchKernelGGL(window_counts, dim3((unsigned)ceil_div(W, 256)), dim3(256), 0, st,
                       d_window_offsets, W, ki, vi);
    F3S_HIP(hipGetLastError());
    // A window's tile count never exceeds W (one tile per block column).
    unsigned end_bit = 1;
    while (end_bit < 32 && ((uint64_t)1 << end_bit) <= (uint64_t)W) ++end_bit;
    size_t bytes = 0;
    F3S_HIP(rocprim::radix_sort_pairs_desc(nullptr, bytes, ki, ko, vi, d_order, (size_t)W, 0,
                                           end_bit, st));
    F3S_TRY(tmp.reserve(bytes));
    // Stable descending sort: equal counts keep ascending window order.
    F3S_HIP(rocprim::radix_sort_pairs_desc(tmp.ptr, bytes, ki, ko, vi, d_order, (size_t)W, 0,
                                           end_bit, st));
    F3S_HIP(hipStreamSynchronize(st));
    return F3S_OK;
}

f3s_status f3s_bsf_stats(const int32_t* d_block_col, const uint16_t* d_tile_mask, int64_t T,
                         int32_t n, int64_t* occ_sum, int64_t* mask_bits, void* stream)
{
    F3S_REQUIRE(T >= 0 && n >= 0, "f3s_bsf_stats: negative size");
    F3S_REQUIRE(occ_sum && mask_bits, "f3s_bsf_stats: NULL output");
    *occ_sum = 0;
    *mask_bits = 0;
    if (T == 0) return F3S_OK;
    F3S_REQUIRE(d_block_col != nullptr, "f3s_bsf_stats: NULL block_col");
    F3S_REQUIRE((((uintptr_t)d_tile_mask) & 15) == 0, "f3s_bsf_stats: tile_mask alignment");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    StreamBuffer out(st);
    F3S_TRY(out.reserve(2 * sizeof(unsigned long long)));
    F3S_HIP(hipMemsetAsync(out.ptr, 0, 2 * sizeof(unsigned long long), st));
    int64_t blocks = ceil_div(T, 256);
    if (blocks > 4096) blocks = 4096;
    hipLaunchKernelGGL(bsf_stats_kernel, dim3((unsigned)blocks), dim3(256), 0, st, d_block_col,
                       d_tile_mask, T, n, reinterpret_cast<unsigned long long*>(out.ptr));
    F3S_HIP(hipGetLastError());
    unsigned long long h[2] = {0, 0};
    F3S_HIP(hipMemcpyAsync(h, out.ptr, sizeof h, hipMemcpyDeviceToHost, st));
    F3S_HIP(hipStreamSynchronize(st));
    *occ_sum = (int64_t)h[0];
    *mask_bits = (int64_t)h[1];
    return F3S_OK;
}

f3s_status f3s_reverse_csr(const int32_t* d_row_ptr, const int32_t* d_col_idx, int32_t n,
                           int64_t nnz, int32_t* d_out_row_ptr, int32_t* d_out_col_idx,
                           void* stream)
{
    F3S_REQUIRE(n >= 0 && nnz >= 0 && nnz <= INT32_MAX, "f3s_reverse_csr: bad size");
    F3S_REQUIRE(n > 0 || nnz == 0, "f3s_reverse_csr: edges without nodes");
    F3S_REQUIRE(d_row_ptr && d_out_row_ptr && (nnz == 0 || (d_col_idx && d_out_col_idx)),
                "f3s_reverse_csr: NULL pointer");
    F3S_TRY(require_device());
    clear_error();
    hipStream_t st = as_stream(stream);
    const size_t words = (size_t)n + (n & 1);
    StreamBuffer buf(st);
    F3S_TRY(buf.reserve(2 * sizeof(int32_t) * words + sizeof(int64_t) * (size_t)(offsets_sum_elems(n) + 1)));
    int32_t* counts = static_cast<int32_t*>(buf.ptr);
    int32_t* used = counts + words;
    int64_t* sums = reinterpret_cast<int64_t*>(used + words);
    if (words)
        hipLaunchKernelGGL(clear_counts, dim3((unsigned)ceil_div(2 * words, 256)), dim3(256), 0, st,
                           counts, (int64_t)(2 * words));
    const dim3 grid((unsigned)ceil_div(nnz, 256));
    if (nnz)
        hipLaunchKernelGGL(column_counts, grid, dim3(256), 0, st, d_col_idx, nnz, n, counts);
    F3S_HIP(hipGetLastError());
    F3S_TRY(counts_to_offsets(counts, d_out_row_ptr, n, sums + 1, sums, st));
    if (nnz) {
        hipLaunchKernelGGL(reverse_fill, grid, dim3(256), 0, st, d_row_ptr, d_col_idx, nnz, n,
                           d_out_row_ptr, used, d_out_col_idx);
        F3S_HIP(hipGetLastError());
    }
    return F3S_OK;
}

}  // extern "C"
