// top_logits.hip -- the k largest logits of every row and the log-sum-exp of the others (sa_top_logits): what a teacher's row
// leaves for a distillation loss.
//
// Values are ordered as (value, lower index first) packed into one 64-bit number (sa_rank_key): all keys of a row differ, so the
// k-th is one element and ties go to the lowest index whatever the order of the work.
//
// One pass over the data.  A workgroup holds a segment of a row in registers.  The k-th largest of its threads' maxima is a bound
// that at least k elements reach and that only k threads' elements can pass: what reaches it are the candidates, a little more
// than k of thousands in ordinary rows, and everything below it goes straight into the log-sum-exp, relative to the bound.  The
// candidates are ranked against each other in LDS.  Where that does not hold -- many ties, NaN, a rest that vanishes
// beside the bound -- the workgroup finds the exact k-th key bit by bit in its registers instead (top_exact).
#include "rows.h"

namespace {

constexpr int kCand = 256;  // candidates a workgroup can hold: k <= 128 of them are kept

struct TopOut {
    float* values;
    long long* ids;
    float* rest;
};

// what a segment leaves for its row, beside its candidates
struct TopPart {
    int count;
    float m, s;  // the others: maximum (or any bound close above it) and the sum of exp((x - m) / T); s = 0: none
};

__device__ __forceinline__ float top_exp(float x, float m, float c) { return x == m ? 1.0f : sa_exp2((x - m) * c); }

// The largest prefix t (most significant bits first) that at least k of the 64 * N keys of this wave reach; stops where few
// enough do.  Uniform over the wave.
template <int N> __device__ __forceinline__ unsigned top_bound(const unsigned (&key)[N], int k) {
    unsigned t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned u = t | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(key[i] >= u));
        if (c >= k) {
            t = u;
            if (c <= k + (k >> 3)) break;
        }
    }
    return t;
}

template <int NT> __device__ __forceinline__ int top_count(int c, int* scratch) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = c;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += scratch[w];
    return s;
}

// Ranks the C <= kCand candidates of the block, writes the first k, leaves the values of the others in `others` in descending order
// (the candidates themselves lie in the order of their arrival, which no result may depend on) and returns the k-th key.
template <int NT>
__device__ __forceinline__ unsigned long long top_rank(const unsigned long long* cand, int C, int k, long row, const TopOut& out,
                                                       unsigned long long* kth, float* others) {
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += NT) {
        const unsigned long long key = cand[c];
        int rank = 0;
        for (int j = 0; j < C; ++j) rank += cand[j] > key;
        if (rank < k) {
            out.values[row * k + rank] = sa_unorder((unsigned)(key >> 32));
            out.ids[row * k + rank] = (long long)(unsigned)~(unsigned)key;
            if (rank == k - 1) *kth = key;
        } else {
            others[rank - k] = sa_unorder((unsigned)(key >> 32));
        }
    }
    __syncthreads();
    return *kth;
}

__device__ __forceinline__ void top_write_rest(float m, float s, float temperature, float* rest) {
    *rest = s == 0.0f ? -INFINITY : m / temperature + logf(s);
}

// A segment of a row: `per` <= NT * NV vectors; nseg == 1: the whole row, and the result.  (The segments of a row are of equal
// length: a short last one would have fewer than k threads with anything, no bound, and take the exact way.)
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void top_segment_kernel(const T* __restrict__ x, SaRows at, int V, int k, int cap,
                                                         float temperature, int nseg, int per, TopOut out,
                                                         unsigned long long* __restrict__ lists, TopPart* __restrict__ parts) {
    constexpr int VEC = SaVec<T>::N;
    __shared__ unsigned long long cand[kCand], kth;
    // one key a thread, or, in rows so short that k threads might not have one, a key an element
    constexpr int KEYS = NV == 1 ? NT * VEC : NT;
    __shared__ unsigned top[KEYS], bound;
    __shared__ int count, counts[NT / 64];
    __shared__ float sums[NT / 64], others[kCand];
    const long row = blockIdx.x / nseg;
    const int seg = blockIdx.x % nseg, tid = threadIdx.x;
    const T* xr = x + at.at(row);
    const int first = seg * per * VEC - sa_lead(xr);  // the segment's first element (may lie before the row)
    const int end = first + per * VEC < V ? first + per * VEC : V;
    const float c = SA_LOG2E / temperature;
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = sa_load_vec(xr, first + (i * NT + tid) * VEC, end);
    const int lo = first < 0 ? 0 : first, valid = end > lo ? end - lo : 0;

    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) mx = fmaxf(mx, sa_element<T>(raw[i], e));
    if constexpr (NV == 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float f = sa_element<T>(raw[0], e);
            top[e * NT + tid] = f == f ? sa_order(f) : 0u;
        }
    } else {
        top[tid] = sa_order(mx);
    }
    if (tid == 0) count = 0;
    __syncthreads();
    if (tid < 64) {
        unsigned key[KEYS / 64];
#pragma unroll
        for (int i = 0; i < KEYS / 64; ++i) key[i] = top[tid + 64 * i];
        const unsigned t = top_bound(key, k);
        if (tid == 0) bound = t;
    }
    __syncthreads();
    const float b = bound <= sa_order(-INFINITY) ? -INFINITY : sa_unorder(bound);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float f = sa_element<T>(raw[i], e);
            if (f >= b) {
                const int v = first + (i * NT + tid) * VEC + e;
                if (v >= 0 && v < end) {
                    const int p = atomicAdd(&count, 1);
                    if (p < kCand) cand[p] = sa_rank_key(f, v);
                }
            } else {
                s += sa_exp2((f - b) * c);
            }
        }
    s = sa_block_sum<NT / 64>(s, sums);
    int C = count;
    float m = b;
    if (C > cap || (C < valid && !(s >= 0x1p-70f))) {
        // exact: the smallest key that min(k, valid) keys reach, bit by bit
        const int want = k < valid ? k : valid;
        unsigned long long K = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long t = K | (1ull << bit);
            int n = 0;
            for (int i = 0; i < NV; ++i)
                for (int e = 0; e < VEC; ++e) {
                    const int v = first + (i * NT + tid) * VEC + e;
                    n += v >= 0 && v < end && sa_rank_key(sa_element<T>(raw[i], e), v) >= t;
                }
            if (top_count<NT>(n, counts) >= want) K = t;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        m = -INFINITY;
        for (int i = 0; i < NV; ++i)
            for (int e = 0; e < VEC; ++e) {
                const int v = first + (i * NT + tid) * VEC + e;
                const float f = sa_element<T>(raw[i], e);
                if (v < 0 || v >= end) continue;
                const unsigned long long key = sa_rank_key(f, v);
                if (key >= K) cand[atomicAdd(&count, 1)] = key;
                else m = fmaxf(m, f);
            }
        m = sa_block_max<NT / 64>(m, sums);
        s = 0.0f;
        for (int i = 0; i < NV; ++i)
            for (int e = 0; e < VEC; ++e) {
                const int v = first + (i * NT + tid) * VEC + e;
                const float f = sa_element<T>(raw[i], e);
                if (v >= 0 && v < end && sa_rank_key(f, v) < K) s += top_exp(f, m, c);
            }
        s = sa_block_sum<NT / 64>(s, sums);
        C = want;
    } else if (C == valid) {
        s = 0.0f;
    }
    if (s == 0.0f) m = -INFINITY;

    if (nseg > 1) {
        if (tid == 0) parts[blockIdx.x] = TopPart{C, m, s};
        __syncthreads();
        for (int i = tid; i < C; i += NT) lists[(size_t)blockIdx.x * cap + i] = cand[i];
        return;
    }
    top_rank<NT>(cand, C, k, row, out, &kth, others);
    // the candidates that were not taken belong to the others
    const float mu = C > k ? others[0] : -INFINITY;
    const float su = sa_block_sum<NT / 64>(tid < C - k ? top_exp(others[tid], mu, c) : 0.0f, sums);
    if (tid == 0) {
        const float M = fmaxf(m, mu);
        top_write_rest(M, s * top_exp(m, M, c) + su * top_exp(mu, M, c), temperature, out.rest + row);
    }
}

// The segments of a row: the same over their candidates, which it reads where the first pass left them.
__global__ __launch_bounds__(256) void top_merge_kernel(const unsigned long long* __restrict__ lists, const TopPart* __restrict__ parts,
                                                        int nseg, int cap, int k, float temperature, TopOut out) {
    constexpr int NT = 256;
    __shared__ unsigned long long cand[kCand], kth;
    __shared__ unsigned top[NT], bound;
    __shared__ int count, counts[NT / 64];
    __shared__ float sums[NT / 64], others[kCand];
    __shared__ unsigned long long total;
    __shared__ int odd;
    const long row = blockIdx.x;
    const int tid = threadIdx.x;
    const float c = SA_LOG2E / temperature;
    lists += (size_t)row * nseg * cap;
    parts += (size_t)row * nseg;
    const int n = nseg * cap;
    unsigned mx = 0;
    for (int i = tid; i < n; i += NT)
        if (i % cap < parts[i / cap].count) {
            const unsigned u = (unsigned)(lists[i] >> 32);
            mx = u > mx ? u : mx;
        }
    top[tid] = mx;
    if (tid == 0) count = 0;
    __syncthreads();
    if (tid < 64) {
        unsigned key[NT / 64];
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) key[i] = top[tid + 64 * i];
        const unsigned t = top_bound(key, k);
        if (tid == 0) bound = t;
    }
    __syncthreads();
    const unsigned b = bound;
    for (int i = tid; i < n; i += NT)
        if (i % cap < parts[i / cap].count) {
            const unsigned long long key = lists[i];
            if ((unsigned)(key >> 32) >= b) {
                const int p = atomicAdd(&count, 1);
                if (p < kCand) cand[p] = key;
            }
        }
    __syncthreads();
    int C = count;
    if (C > kCand) {
        unsigned long long K = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long t = K | (1ull << bit);
            int r = 0;
            for (int i = tid; i < n; i += NT) r += i % cap < parts[i / cap].count && lists[i] >= t;
            if (top_count<NT>(r, counts) >= k) K = t;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        for (int i = tid; i < n; i += NT)
            if (i % cap < parts[i / cap].count && lists[i] >= K) cand[atomicAdd(&count, 1)] = lists[i];
        C = k;
    }
    const unsigned long long last = top_rank<NT>(cand, C, k, row, out, &kth, others);
    float m = -INFINITY;
    // the reference is the largest TERM, not the largest bound: a segment's sum may be as small as 2^-70 of its bound
    for (int i = tid; i < nseg; i += NT)
        if (parts[i].s != 0.0f) m = fmaxf(m, parts[i].m + sa_log2(parts[i].s) / c);
    for (int i = tid; i < n; i += NT)
        if (i % cap < parts[i / cap].count && lists[i] < last) m = fmaxf(m, sa_unorder((unsigned)(lists[i] >> 32)));
    m = sa_block_max<NT / 64>(m, sums);
    float s = 0.0f;
    for (int i = tid; i < nseg; i += NT)
        if (parts[i].s != 0.0f) s += parts[i].s * top_exp(parts[i].m, m, c);
    s = sa_block_sum<NT / 64>(s, sums);
    // The lists are in the order of arrival: their terms (0 .. 1) are summed as integers of 2^-32, the same in any order.
    if (tid == 0) { total = 0; odd = 0; }
    __syncthreads();
    unsigned long long u = 0;
    for (int i = tid; i < n; i += NT)
        if (i % cap < parts[i / cap].count && lists[i] < last) {
            const float e = top_exp(sa_unorder((unsigned)(lists[i] >> 32)), m, c);
            if (e == e) u += (unsigned long long)(e * 0x1p32f);
            else odd = 1;
        }
    if (u) atomicAdd(&total, u);
    __syncthreads();
    s += odd ? NAN : (float)total * 0x1p-32f;
    if (tid == 0) top_write_rest(m, s, temperature, out.rest + row);
}

// Short rows (V <= 128): a wave each, every element ranked against all others.
template <typename T>
__global__ __launch_bounds__(256) void top_short_kernel(const T* __restrict__ x, SaRows at, long rows, int V, int k,
                                                        float temperature, TopOut out) {
    __shared__ unsigned long long keys[4][128];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long row = (long)blockIdx.x * 4 + w;
    if (row >= rows) return;  // (no barrier below: a wave's LDS accesses are in order)
    const T* xr = x + at.at(row);
    const float c = SA_LOG2E / temperature;
    float f[2];
    unsigned long long key[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int v = lane + 64 * i;
        f[i] = v < V ? sa_widen(xr[v]) : -INFINITY;
        key[i] = v < V ? sa_rank_key(f[i], v) : 0;
        keys[w][v] = key[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    int rank[2] = {0, 0};
    for (int j = 0; j < V; ++j) {
        const unsigned long long o = keys[w][j];
        rank[0] += o > key[0];
        rank[1] += o > key[1];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int v = lane + 64 * i;
        if (v >= V) continue;
        if (rank[i] < k) {
            out.values[row * k + rank[i]] = f[i];
            out.ids[row * k + rank[i]] = v;
        } else {
            m = fmaxf(m, f[i]);
        }
    }
    m = sa_wave_max(m);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < V && rank[i] >= k) s += top_exp(f[i], m, c);
    s = sa_wave_sum(s);
    if (lane == 0) top_write_rest(m, s, temperature, out.rest + row);
}

struct TopPlan {
    int nv, nseg, per, cap;  // vectors a thread, segments a row, vectors a segment, candidates a segment may leave
};
TopPlan top_plan(int V, int k, int dtype) {
    const int vec = dtype == SA_F32 ? 4 : 8, vectors = (V + vec - 1 + vec - 1) / vec;  // the longest row, with its lead
    TopPlan p;
    p.nv = vectors <= 256 ? 1 : vectors <= 512 ? 2 : vectors <= 1024 ? 4 : 8;
    p.nseg = (vectors + 256 * p.nv - 1) / (256 * p.nv);
    p.per = (vectors + p.nseg - 1) / p.nseg;
    p.nseg = (vectors + p.per - 1) / p.per;
    p.cap = k + k / 2 + 32;
    return p;
}
size_t top_bytes(long rows, const TopPlan& p) {
    return p.nseg == 1 ? 0
                       : sa_align_up((size_t)rows * p.nseg * sizeof(TopPart), 256) +
                             (size_t)rows * p.nseg * p.cap * sizeof(unsigned long long);
}

template <typename T>
void top_launch(const void* x, const SaRows& at, long rows, int V, int k, float temperature, const TopOut& out,
                const TopPlan& p, char* ws, hipStream_t stream) {
    const T* xt = (const T*)x;
    if (V <= 128) {
        hipLaunchKernelGGL((top_short_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, xt, at, rows, V, k,
                           temperature, out);
        return;
    }
    TopPart* parts = (TopPart*)ws;
    unsigned long long* lists = (unsigned long long*)(ws + sa_align_up((size_t)rows * p.nseg * sizeof(TopPart), 256));
    const int cap = p.nseg == 1 ? kCand : p.cap;
    const dim3 grid((unsigned)(rows * p.nseg)), block(256);
#define TOP_LAUNCH(NV)                                                                                                     \
    hipLaunchKernelGGL((top_segment_kernel<T, 256, NV>), grid, block, 0, stream, xt, at, V, k, cap, temperature, p.nseg, p.per, out, \
                       lists, parts)
    if (p.nv == 1) TOP_LAUNCH(1);
    else if (p.nv == 2) TOP_LAUNCH(2);
    else if (p.nv == 4) TOP_LAUNCH(4);
    else TOP_LAUNCH(8);
#undef TOP_LAUNCH
    if (p.nseg > 1)
        hipLaunchKernelGGL(top_merge_kernel, dim3((unsigned)rows), dim3(256), 0, stream, (const unsigned long long*)lists,
                           (const TopPart*)parts, p.nseg, p.cap, k, temperature, out);
}

bool top_ok(long rows, int V, int k, int dtype) {
    return rows >= 0 && sa_rows_ok(dtype, V) && k >= 1 && k <= V && k <= SA_TOP_MAX &&
           (size_t)rows * (size_t)top_plan(V, k, dtype).nseg <= 0x7fffffffu;
}

}  // namespace

extern "C" size_t sa_top_logits_workspace_bytes(long rows, int V, int k, int dtype) {
    return top_ok(rows, V, k, dtype) ? top_bytes(rows, top_plan(V, k, dtype)) : 0;
}

extern "C" ctcStatus_t sa_top_logits(const void* x, long ld_outer, long ld_inner, int n_inner, int dtype, long rows, int V,
                                     int k, float temperature, float* values, long long* ids, float* rest, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    SA_CLEAR_ERR();
    if (!top_ok(rows, V, k, dtype) || n_inner < 1 || !(temperature > 0.f) || !(temperature < INFINITY))
        return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const TopPlan p = top_plan(V, k, dtype);
    if (!x || !values || !ids || !rest || (top_bytes(rows, p) && (!workspace || workspace_bytes < top_bytes(rows, p))))
        return CTC_STATUS_INVALID_VALUE;
    const SaRows at{ld_outer, ld_inner, n_inner};
    const TopOut out{values, ids, rest};
    if (dtype == SA_F32) top_launch<float>(x, at, rows, V, k, temperature, out, p, (char*)workspace, (hipStream_t)stream);
    else if (dtype == SA_BF16) top_launch<SaBf16>(x, at, rows, V, k, temperature, out, p, (char*)workspace, (hipStream_t)stream);
    else top_launch<SaF16>(x, at, rows, V, k, temperature, out, p, (char*)workspace, (hipStream_t)stream);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
