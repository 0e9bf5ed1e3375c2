// constrain.hip -- penalties for repeated tokens, biases and grammar masks on output rows, and the token that is left
// (sa_logits_constrain, sa_logits_pick; the arithmetic is stated in include/speech_amd.h).
//
// A workgroup takes a segment of a row.  What the history and the bias list say about the segment's tokens is gathered in LDS
// first, one 32-bit word a token: the low half counts the token in the history, the high half holds 1 + the position of the
// last bias entry of that token (hence the limit of 65535 on both lists).  Integer maxima and sums: the order in which the
// lanes arrive does not matter.  The row itself is read once.
#include "rows.h"

namespace {

constexpr int kConThreads = 256, kConEach = 16, kConSeg = kConThreads * kConEach;

struct PickPart {  // what a segment leaves for its row: the best token, the maximum and the sum of exp(x - maximum)
    unsigned long long key;
    float m, s;
};

// exp(x - m) where equal infinities count as equal (a bias of +inf forces its token)
__device__ __forceinline__ float con_exp(float x, float m) { return x == m ? 1.0f : sa_exp2((x - m) * SA_LOG2E); }

template <typename T>
__device__ __forceinline__ float con_value(T raw, unsigned word, bool allowed, float r, float p, float f, const float* bias) {
#pragma clang fp contract(off)  // every step is rounded as the formula is written: the token must not depend on a fused step
    float x = sa_widen(raw);
    const unsigned c = word & 0xffffu, b = word >> 16;
    if (c) {
        x = x > 0.0f ? x / r : x * r;
        x = x - (float)c * f;
        x = x - p;
    }
    if (b) x = x + bias[b - 1];
    return allowed ? x : -INFINITY;
}

// The two lists of `row`, for the tokens [v0, v0 + n): every thread of the block calls it.
__device__ __forceinline__ void con_lists(unsigned* words, const saConstraints& C, int row, int v0, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) words[i] = 0;
    __syncthreads();
    if (C.bias_ids) {
        const long long* ids = C.bias_ids + (long)row * C.bias_ld;
        for (int j = threadIdx.x; j < C.n_bias; j += blockDim.x) {
            const unsigned long long d = (unsigned long long)(ids[j] - v0);
            if (d < (unsigned long long)n) atomicMax(&words[d], (unsigned)(j + 1) << 16);
        }
        __syncthreads();
    }
    if (C.history) {
        const long long* h = C.history + (long)row * C.history_ld;
        int len = C.lengths ? C.lengths[row] : C.history_len;
        len = len < 0 ? 0 : (len > C.history_len ? C.history_len : len);
        for (int i = threadIdx.x; i < len; i += blockDim.x) {
            const unsigned long long d = (unsigned long long)(h[i] - v0);
            if (d < (unsigned long long)n) atomicAdd(&words[d], 1u);
        }
    }
    __syncthreads();
}

template <typename T, bool PICK>
__global__ __launch_bounds__(kConThreads) void constrain_kernel(const T* __restrict__ x, long ldx, T* y, long ldy, int V,
                                                                int nseg, saConstraints C, PickPart* __restrict__ part,
                                                                long long* __restrict__ tokens, float* __restrict__ logp) {
    __shared__ unsigned words[kConSeg];
    __shared__ float scratch[kConThreads / 64];
    __shared__ unsigned long long best[kConThreads / 64];
    const int row = blockIdx.x / nseg, seg = blockIdx.x % nseg, tid = threadIdx.x;
    const int v0 = seg * kConSeg, n = V - v0 < kConSeg ? V - v0 : kConSeg;
    con_lists(words, C, row, v0, n);
    const float r = C.repetition ? C.repetition[row] : C.repetition_all;
    const float p = C.presence ? C.presence[row] : C.presence_all;
    const float f = C.frequency ? C.frequency[row] : C.frequency_all;
    const float* bias = C.bias_values + (long)row * C.bias_ld;
    const unsigned* mask = nullptr;
    if (C.mask) {
        const int state = C.states ? C.states[row] : row;
        if (state >= 0 && state < C.n_states) mask = C.mask + (long)state * C.mask_ld;
    }
    const T* xr = x + (long)row * ldx + v0;
    float val[kConEach];
    unsigned long long key = 0;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kConEach; ++j) {
        const int i = tid + j * kConThreads;
        val[j] = -INFINITY;
        if (i < n) {
            const int v = v0 + i;
            const bool allowed = !mask || ((mask[v >> 5] >> (v & 31)) & 1u);
            val[j] = con_value(xr[i], words[i], allowed, r, p, f, bias);
            if (PICK) {
                const unsigned long long k = sa_rank_key(val[j], v);
                key = k > key ? k : key;
                m = fmaxf(m, val[j]);
            } else {
                y[(long)row * ldy + v] = sa_narrow<T>(val[j]);
            }
        }
    }
    if (!PICK) return;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor(key, o, 64);
        key = other > key ? other : key;
    }
    if ((tid & 63) == 0) best[tid >> 6] = key;
    m = sa_block_max<kConThreads / 64>(m, scratch);  // (its barriers also publish `best`)
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kConEach; ++j)
        if (tid + j * kConThreads < n) s += con_exp(val[j], m);
    s = sa_block_sum<kConThreads / 64>(s, scratch);
    if (tid == 0) {
        for (int w = 0; w < kConThreads / 64; ++w) key = best[w] > key ? best[w] : key;
        if (nseg == 1) {
            const bool none = (unsigned)(key >> 32) == sa_order(-INFINITY);
            tokens[row] = none ? -1 : (long long)(unsigned)~(unsigned)key;
            logp[row] = none ? -INFINITY : -logf(s);
        } else {
            part[blockIdx.x] = PickPart{key, m, s};
        }
    }
}

// the segments of a row, in their order, by one wave
__global__ __launch_bounds__(64) void pick_join_kernel(const PickPart* __restrict__ part, int nseg, long long* __restrict__ tokens,
                                                       float* __restrict__ logp) {
    const PickPart* P = part + (long)blockIdx.x * nseg;
    unsigned long long key = 0;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < nseg; i += 64) {
        key = P[i].key > key ? P[i].key : key;
        m = fmaxf(m, P[i].m);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor(key, o, 64);
        key = other > key ? other : key;
    }
    m = sa_wave_max(m);
    float s = 0.f;
    for (int i = threadIdx.x; i < nseg; i += 64) s += P[i].s * con_exp(P[i].m, m);
    s = sa_wave_sum(s);
    if (threadIdx.x == 0) {
        const bool none = (unsigned)(key >> 32) == sa_order(-INFINITY);
        tokens[blockIdx.x] = none ? -1 : (long long)(unsigned)~(unsigned)key;
        logp[blockIdx.x] = none ? -INFINITY : -logf(s);
    }
}

int con_segments(int V) { return (V + kConSeg - 1) / kConSeg; }

bool con_ok(const saConstraints* c, int rows, int V) {
    if (!c || c->history_len < 0 || c->history_len > SA_LIST_MAX || c->n_bias < 0 || c->n_bias > SA_LIST_MAX) return false;
    if (c->history_len > 0 && (!c->history || c->history_ld < 0)) return false;
    if (c->n_bias > 0 && (!c->bias_ids || !c->bias_values || c->bias_ld < 0)) return false;
    if (c->mask && (c->n_states < 1 || c->mask_ld < (V + 31) / 32 || (!c->states && c->n_states < rows))) return false;
    return true;
}

// what the kernels test is the pointer alone
saConstraints con_used(const saConstraints& c) {
    saConstraints u = c;
    if (u.history_len == 0) u.history = nullptr;
    if (u.n_bias == 0) u.bias_ids = nullptr;
    return u;
}

template <bool PICK>
void con_launch(const void* x, long ldx, int dtype, void* y, long ldy, int rows, int V, const saConstraints& c, PickPart* part,
                long long* tokens, float* logp, hipStream_t stream) {
    const saConstraints C = con_used(c);
    const int nseg = con_segments(V);
    const dim3 grid((unsigned)((size_t)rows * nseg)), block(kConThreads);
    if (dtype == SA_F32)
        hipLaunchKernelGGL((constrain_kernel<float, PICK>), grid, block, 0, stream, (const float*)x, ldx, (float*)y, ldy, V, nseg, C,
                           part, tokens, logp);
    else if (dtype == SA_BF16)
        hipLaunchKernelGGL((constrain_kernel<SaBf16, PICK>), grid, block, 0, stream, (const SaBf16*)x, ldx, (SaBf16*)y, ldy, V,
                           nseg, C, part, tokens, logp);
    else
        hipLaunchKernelGGL((constrain_kernel<SaF16, PICK>), grid, block, 0, stream, (const SaF16*)x, ldx, (SaF16*)y, ldy, V, nseg,
                           C, part, tokens, logp);
}

}  // namespace

extern "C" ctcStatus_t sa_logits_constrain(const void* x, long ldx, int dtype, void* y, long ldy, int rows, int V,
                                           const saConstraints* c, void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || !sa_rows_ok(dtype, V) || !con_ok(c, rows, V)) return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    if (!x || !y || (size_t)rows * con_segments(V) > 0x7fffffffu) return CTC_STATUS_INVALID_VALUE;
    con_launch<false>(x, ldx, dtype, y, ldy, rows, V, *c, nullptr, nullptr, nullptr, (hipStream_t)stream);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}

extern "C" size_t sa_logits_pick_workspace_bytes(int rows, int V) {
    if (rows < 1 || V < 1 || V > SA_VOCAB_MAX || con_segments(V) == 1) return 0;
    return (size_t)rows * con_segments(V) * sizeof(PickPart);
}

extern "C" ctcStatus_t sa_logits_pick(const void* x, long ldx, int dtype, int rows, int V, const saConstraints* c,
                                      long long* d_tokens, float* d_logp, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || !sa_rows_ok(dtype, V) || !con_ok(c, rows, V)) return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const size_t need = sa_logits_pick_workspace_bytes(rows, V);
    if (!x || !d_tokens || !d_logp || (need && (!workspace || workspace_bytes < need)) ||
        (size_t)rows * con_segments(V) > 0x7fffffffu)
        return CTC_STATUS_INVALID_VALUE;
    con_launch<true>(x, ldx, dtype, nullptr, 0, rows, V, *c, (PickPart*)workspace, d_tokens, d_logp, (hipStream_t)stream);
    if (need)
        hipLaunchKernelGGL(pick_join_kernel, dim3(rows), dim3(64), 0, (hipStream_t)stream, (const PickPart*)workspace,
                           con_segments(V), d_tokens, d_logp);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
