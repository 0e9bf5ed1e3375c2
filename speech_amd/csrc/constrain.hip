// constrain.hip -- penalties for repeated tokens, biases and grammar masks on output rows, and the token that is left
// (sa_logits_constrain, sa_logits_pick; the arithmetic is stated in include/speech_amd.h).
//
// A workgroup takes a segment of a row and reads it once, as 16-byte vectors, into registers.  Meanwhile the history and the bias
// list are gathered in LDS, one 32-bit word a token of the segment: the low half counts the token in the history, the high half
// holds 1 + the position of the last bias entry of that token (hence the limit of 65535 on both lists).  Integer maxima and
// sums: the order in which the lanes arrive does not matter.  The few tokens that are found there are collected, and their final
// logits -- the division and the other steps that most tokens do not need -- take the place of their words.  Then every element is
// either its logit or its word, masked, and stored or reduced.
#include "rows.h"

namespace {

struct PickPart {  // what a segment leaves for its row: the best token, the maximum and the sum of exp(x - maximum)
    unsigned long long key;
    float m, s;
};

// exp(x - m) where equal infinities count as equal (a bias of +inf forces its token)
__device__ __forceinline__ float con_exp(float x, float m) { return x == m ? 1.0f : sa_exp2((x - m) * SA_LOG2E); }

__device__ __forceinline__ float con_value(float x, unsigned word, float r, float p, float f, const float* bias) {
#pragma clang fp contract(off)  // every step is rounded as the formula is written: the token must not depend on a fused step
    const unsigned c = word & 0xffffu, b = word >> 16;
    if (c) {
        x = x > 0.0f ? x / r : x * r;
        x = x - (float)c * f;
        x = x - p;
    }
    if (b) x = x + bias[b - 1];
    return x;
}

// bits v0 .. v0 + VEC - 1 of a mask row (bits of tokens outside [0, V) are not looked at by anybody)
template <int VEC> __device__ __forceinline__ unsigned con_allowed(const unsigned* __restrict__ mask, int v0, int V) {
    const int lo = v0 < 0 ? 0 : v0 >> 5, last = (V - 1) >> 5, hi = (v0 + VEC - 1) >> 5;
    const unsigned a = mask[lo > last ? last : lo], b = mask[hi < 0 ? 0 : hi > last ? last : hi];
    if (v0 < 0) return a << -v0;
    return (unsigned)(((((unsigned long long)b) << 32 | a)) >> (v0 & 31));
}

template <typename T, int NV, bool PICK>
__global__ __launch_bounds__(256) void constrain_kernel(const T* x, long ldx, T* y /* may be x */, long ldy, int V, int nseg, int per,
                                                        saConstraints C, PickPart* __restrict__ part, long long* __restrict__ tokens,
                                                        float* __restrict__ logp) {
    constexpr int VEC = SaVec<T>::N, NT = 256, SEG = NT * NV * VEC;
    extern __shared__ unsigned words[];  // SEG words, then SEG positions (16 bits); nothing where there are no lists
    __shared__ int found;
    __shared__ float scratch[NT / 64];
    __shared__ unsigned long long best[NT / 64];
    const int row = blockIdx.x / nseg, seg = blockIdx.x % nseg, tid = threadIdx.x;
    const T* xr = x + (long)row * ldx;
    const int first = seg * per * VEC - sa_lead(xr), end = first + per * VEC < V ? first + per * VEC : V;
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = sa_load_vec(xr, first + (i * NT + tid) * VEC, end);
    const unsigned* mask = nullptr;
    if (C.mask) {
        const int state = C.states ? C.states[row] : row;
        if (state >= 0 && state < C.n_states) mask = C.mask + (long)state * C.mask_ld;
    }
    const bool lists = C.history || C.bias_ids;
    if (lists) {
        sa_u16* places = (sa_u16*)(words + SEG);
        const float r = C.repetition ? C.repetition[row] : C.repetition_all;
        const float p = C.presence ? C.presence[row] : C.presence_all;
        const float f = C.frequency ? C.frequency[row] : C.frequency_all;
        const float* bias = C.bias_values + (long)row * C.bias_ld;
        int len = 0;
        if (C.history) {
            len = C.lengths ? C.lengths[row] : C.history_len;
            len = len < 0 ? 0 : (len > C.history_len ? C.history_len : len);
        }
        uint4* clear = (uint4*)words;
#pragma unroll
        for (int i = 0; i < SEG / 4 / NT; ++i) clear[i * NT + tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) found = 0;
        // (a token t of a list is the segment's when `first` <= t < `end`; t >= 0 keeps what lies before the row out; the last
        // segment of a row that starts on a boundary may be empty, and begin behind the row's end)
        const unsigned long long n = end > first ? (unsigned long long)(end - first) : 0ull;
        __syncthreads();
        if (C.bias_ids) {
            const long long* ids = C.bias_ids + (long)row * C.bias_ld;
            for (int j = tid; j < C.n_bias; j += NT) {
                const long long t = ids[j];
                const unsigned long long d = (unsigned long long)(t - first);
                if (t >= 0 && d < n && atomicMax(&words[d], (unsigned)(j + 1) << 16) == 0) places[atomicAdd(&found, 1)] = (sa_u16)d;
            }
            __syncthreads();
        }
        if (len > 0) {
            const long long* h = C.history + (long)row * C.history_ld;
#pragma unroll 4
            for (int i = tid; i < len; i += NT) {
                const long long t = h[i];
                const unsigned long long d = (unsigned long long)(t - first);
                if (t >= 0 && d < n && atomicAdd(&words[d], 1u) == 0) places[atomicAdd(&found, 1)] = (sa_u16)d;
            }
        }
        __syncthreads();
        for (int i = tid; i < found; i += NT) {
            const int d = places[i];
            const unsigned u = __builtin_bit_cast(unsigned, con_value(sa_widen(xr[first + d]), words[d], r, p, f, bias));
            words[d] = u ? u : 0x80000000u;  // (0 marks a token that is in no list)
        }
        __syncthreads();
    }
    T* yr = PICK ? nullptr : y + (long)row * ldy;
    const bool aligned = !PICK && sa_lead(yr) == sa_lead(xr);
    unsigned long long key = 0;
    float m = -INFINITY, val[PICK ? NV * VEC : VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int q = i * NT + tid, v0 = first + q * VEC;
        if (v0 >= end) {
            if (PICK)
#pragma unroll
                for (int e = 0; e < VEC; ++e) val[i * VEC + e] = -INFINITY;
            continue;
        }
        float* g = val + (PICK ? i * VEC : 0);
        const unsigned allowed = mask ? con_allowed<VEC>(mask, v0, V) : ~0u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            g[e] = sa_element<T>(raw[i], e);
            if (lists) {
                const unsigned w = words[q * VEC + e];
                g[e] = w ? __builtin_bit_cast(float, w) : g[e];
            }
            g[e] = (allowed >> e) & 1u ? g[e] : -INFINITY;
        }
        if constexpr (PICK) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (v0 + e >= 0 && v0 + e < end) {
                    const unsigned long long k = sa_rank_key(g[e], v0 + e);
                    key = k > key ? k : key;
                    m = fmaxf(m, g[e]);
                } else {
                    g[e] = -INFINITY;
                }
            }
        } else {
            sa_store_vec<T>(yr, v0, end, g, aligned);
        }
    }
    if constexpr (PICK) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor(key, o, 64);
            key = other > key ? other : key;
        }
        if ((tid & 63) == 0) best[tid >> 6] = key;
        m = sa_block_max<NT / 64>(m, scratch);  // (its barriers also publish `best`)
        float s = 0.0f;
        if (m > -INFINITY) {  // (else every exponential would be that of equal infinities; nothing is left anyway)
#pragma unroll
            for (int i = 0; i < NV * VEC; ++i) s += con_exp(val[i], m);
        } else {
#pragma unroll
            for (int i = 0; i < NV * VEC; ++i) s += val[i] == val[i] ? 0.0f : NAN;
        }
        s = sa_block_sum<NT / 64>(s, scratch);
        if (tid == 0) {
            for (int w = 0; w < NT / 64; ++w) key = best[w] > key ? best[w] : key;
            if (nseg == 1) {
                const bool none = (unsigned)(key >> 32) == sa_order(-INFINITY);
                tokens[row] = none ? -1 : (long long)(unsigned)~(unsigned)key;
                logp[row] = none ? -INFINITY : -logf(s);
            } else {
                part[blockIdx.x] = PickPart{key, m, s};
            }
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
    for (int i = threadIdx.x; i < nseg; i += 64)
        if (P[i].m > -INFINITY || P[i].s != 0.0f) s += P[i].s * con_exp(P[i].m, m);
    s = sa_wave_sum(s);
    if (threadIdx.x == 0) {
        const bool none = (unsigned)(key >> 32) == sa_order(-INFINITY);
        tokens[blockIdx.x] = none ? -1 : (long long)(unsigned)~(unsigned)key;
        logp[blockIdx.x] = none ? -INFINITY : -logf(s);
    }
}

// Vectors a thread, segments a row, vectors a segment.  Segments as long as the registers and 48 KB of LDS allow -- each reads
// the lists of its row again -- unless that leaves CUs without work; a row that one workgroup can hold is not split where that
// would cost pick a second launch.
struct ConPlan { int nv, nseg, per; };
ConPlan con_plan(int rows, int V, int dtype, bool pick) {
    const int vec = dtype == SA_F32 ? 4 : 8, most = dtype == SA_F32 ? 8 : 4, vectors = (V + 2 * vec - 2) / vec;
    ConPlan p{1, 1, 0};
    while (p.nv < most && 256 * p.nv < vectors &&
           ((pick && vectors <= 256 * most) || (long)rows * ((vectors + 512 * p.nv - 1) / (512 * p.nv)) >= 512))
        p.nv *= 2;
    p.nseg = (vectors + 256 * p.nv - 1) / (256 * p.nv);
    p.per = (vectors + p.nseg - 1) / p.nseg;
    p.nseg = (vectors + p.per - 1) / p.per;
    return p;
}

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

template <typename T, bool PICK>
void con_launch(const void* x, long ldx, void* y, long ldy, int rows, int V, const ConPlan& p, const saConstraints& c,
                PickPart* part, long long* tokens, float* logp, hipStream_t stream) {
    const saConstraints C = con_used(c);
    const dim3 grid((unsigned)((size_t)rows * p.nseg)), block(256);
    const size_t smem = C.history || C.bias_ids ? (size_t)256 * p.nv * SaVec<T>::N * 6 : 0;
#define CON_LAUNCH(NV)                                                                                                        \
    hipLaunchKernelGGL((constrain_kernel<T, NV, PICK>), grid, block, smem, stream, (const T*)x, ldx, (T*)y, ldy, V, p.nseg, p.per, \
                       C, part, tokens, logp)
    if (p.nv == 1) CON_LAUNCH(1);
    else if (p.nv == 2) CON_LAUNCH(2);
    else if (p.nv == 4) CON_LAUNCH(4);
    else if constexpr (sizeof(T) == 4) CON_LAUNCH(8);
#undef CON_LAUNCH
}

template <bool PICK>
void con_run(const void* x, long ldx, int dtype, void* y, long ldy, int rows, int V, const ConPlan& p, const saConstraints& c,
             PickPart* part, long long* tokens, float* logp, hipStream_t stream) {
    if (dtype == SA_F32) con_launch<float, PICK>(x, ldx, y, ldy, rows, V, p, c, part, tokens, logp, stream);
    else if (dtype == SA_BF16) con_launch<SaBf16, PICK>(x, ldx, y, ldy, rows, V, p, c, part, tokens, logp, stream);
    else con_launch<SaF16, PICK>(x, ldx, y, ldy, rows, V, p, c, part, tokens, logp, stream);
}

}  // namespace

extern "C" ctcStatus_t sa_logits_constrain(const void* x, long ldx, int dtype, void* y, long ldy, int rows, int V,
                                           const saConstraints* c, void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || !sa_rows_ok(dtype, V) || !con_ok(c, rows, V)) return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const ConPlan p = con_plan(rows, V, dtype, false);
    if (!x || !y || (size_t)rows * p.nseg > 0x7fffffffu) return CTC_STATUS_INVALID_VALUE;
    con_run<false>(x, ldx, dtype, y, ldy, rows, V, p, *c, nullptr, nullptr, nullptr, (hipStream_t)stream);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}

extern "C" size_t sa_logits_pick_workspace_bytes(int rows, int V, int dtype) {
    if (rows < 1 || !sa_rows_ok(dtype, V)) return 0;
    const ConPlan p = con_plan(rows, V, dtype, true);
    return p.nseg == 1 ? 0 : (size_t)rows * p.nseg * sizeof(PickPart);
}

extern "C" ctcStatus_t sa_logits_pick(const void* x, long ldx, int dtype, int rows, int V, const saConstraints* c,
                                      long long* d_tokens, float* d_logp, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || !sa_rows_ok(dtype, V) || !con_ok(c, rows, V)) return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const ConPlan p = con_plan(rows, V, dtype, true);
    const size_t need = sa_logits_pick_workspace_bytes(rows, V, dtype);
    if (!x || !d_tokens || !d_logp || (need && (!workspace || workspace_bytes < need)) || (size_t)rows * p.nseg > 0x7fffffffu)
        return CTC_STATUS_INVALID_VALUE;
    con_run<true>(x, ldx, dtype, nullptr, 0, rows, V, p, *c, (PickPart*)workspace, d_tokens, d_logp, (hipStream_t)stream);
    if (need)
        hipLaunchKernelGGL(pick_join_kernel, dim3(rows), dim3(64), 0, (hipStream_t)stream, (const PickPart*)workspace, p.nseg,
                           d_tokens, d_logp);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
