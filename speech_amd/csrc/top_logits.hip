// top_logits.hip -- the k largest logits of every row and the log-sum-exp of the others (sa_top_logits): what a teacher's row
// leaves for a distillation loss.
//
// Values are ordered as (value, lower index first) packed into one 64-bit number (sa_rank_key): all keys of a row differ, so the
// k-th is one element and ties go to the lowest index whatever the order of the work.
#include "rows.h"

namespace {

constexpr int kTopThreads = 256;

// A workgroup per row; entry j is the largest key below entry j - 1.
template <typename T>
__global__ __launch_bounds__(kTopThreads) void top_scan_kernel(const T* __restrict__ x, SaRows at, int V, int k, float temperature,
                                                               float* __restrict__ values, long long* __restrict__ ids,
                                                               float* __restrict__ rest) {
    __shared__ unsigned long long best[kTopThreads / 64];
    __shared__ float scratch[kTopThreads / 64];
    const long row = blockIdx.x;
    const T* xr = x + at.at(row);
    const float c = SA_LOG2E / temperature;
    unsigned long long last = ~0ull;
    for (int j = 0; j < k; ++j) {
        unsigned long long key = 0;
        for (int v = threadIdx.x; v < V; v += kTopThreads) {
            const unsigned long long q = sa_rank_key(sa_widen(xr[v]), v);
            if (q < last && q > key) key = q;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor(key, o, 64);
            key = other > key ? other : key;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = key;
        __syncthreads();
        for (int w = 0; w < kTopThreads / 64; ++w) key = best[w] > key ? best[w] : key;
        last = key;
        if (threadIdx.x == 0) {
            values[row * k + j] = sa_unorder((unsigned)(key >> 32));
            ids[row * k + j] = (long long)(unsigned)~(unsigned)key;
        }
    }
    float m = -INFINITY, s = 0.f;
    for (int v = threadIdx.x; v < V; v += kTopThreads) {
        const float f = sa_widen(xr[v]);
        if (sa_rank_key(f, v) < last) m = fmaxf(m, f);
    }
    m = sa_block_max<kTopThreads / 64>(m, scratch);
    for (int v = threadIdx.x; v < V; v += kTopThreads) {
        const float f = sa_widen(xr[v]);
        if (sa_rank_key(f, v) < last) s += f == m ? 1.0f : sa_exp2((f - m) * c);
    }
    s = sa_block_sum<kTopThreads / 64>(s, scratch);
    if (threadIdx.x == 0) rest[row] = (s > 0.f || s != s) ? m / temperature + logf(s) : -INFINITY;
}

}  // namespace

extern "C" size_t sa_top_logits_workspace_bytes(long rows, int V, int k, int dtype) { return 0; }

extern "C" ctcStatus_t sa_top_logits(const void* x, long ld_outer, long ld_inner, int n_inner, int dtype, long rows, int V,
                                     int k, float temperature, float* values, long long* ids, float* rest, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || rows > 0x7fffffffL || n_inner < 1 || !sa_rows_ok(dtype, V) || k < 1 || k > V || k > SA_TOP_MAX ||
        !(temperature > 0.f) || !(temperature < INFINITY))
        return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    if (!x || !values || !ids || !rest) return CTC_STATUS_INVALID_VALUE;
    const SaRows at{ld_outer, ld_inner, n_inner};
    const dim3 grid((unsigned)rows), block(kTopThreads);
    if (dtype == SA_F32)
        hipLaunchKernelGGL((top_scan_kernel<float>), grid, block, 0, (hipStream_t)stream, (const float*)x, at, V, k, temperature, values,
                           ids, rest);
    else if (dtype == SA_BF16)
        hipLaunchKernelGGL((top_scan_kernel<SaBf16>), grid, block, 0, (hipStream_t)stream, (const SaBf16*)x, at, V, k, temperature, values,
                           ids, rest);
    else
        hipLaunchKernelGGL((top_scan_kernel<SaF16>), grid, block, 0, (hipStream_t)stream, (const SaF16*)x, at, V, k, temperature, values,
                           ids, rest);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
