// constrain.hip -- penalties for repeated tokens, biases and grammar masks on output rows, and the token that is left
// (sa_logits_constrain, sa_logits_pick; the arithmetic is stated in include/speech_amd.h).
//
// A workgroup takes a segment of a row and reads it once, as 16-byte vectors, into registers.  Meanwhile the history and the bias
// list are gathered in LDS, one 32-bit word a token of the segment: the low half counts the token in the history, the high half
// holds 1 + the position of the last bias entry of that token (hence the limit of 65535 on both lists).  Integer maxima and
// sums: the order in which the lanes arrive does not matter.  The few tokens that are found there are collected, and their final
// logits -- the division and the other steps that most tokens do not need -- take the place of their words.  Then every element is
// either its logit or its word, masked, and stored or reduced.
//
// Large batches are bound by memory (256 x 131072 f32 with 4096 tokens of history, constrained: 68 us, 4.0 TB/s, where the bytes
// alone take 54), small ones by the chain list -> LDS -> word -> logit, once per workgroup and a few of them on every CU (pick,
// 64 x 50021 bf16 with 2048 tokens of history: 11 us, and 4 for the join of its segments).
#include "rows.h"

namespace {

// What a wave leaves for its segment, and a segment for its row: the order of the best value (sa_order: NaN above all) and the
// lowest token that has it, the largest number and the sum of exp(x - m).  m = -inf: no numbers.
struct PickPart {
    unsigned best;
    int token;
    float m, s;
};
__device__ __forceinline__ void pick_better(PickPart& a, unsigned best, int token) {
    if (best > a.best || (best == a.best && token < a.token)) { a.best = best; a.token = token; }
}
__device__ __forceinline__ void pick_write(const PickPart& a, long long* token, float* logp) {
    const bool none = a.best <= sa_order(-INFINITY);
    *token = none ? -1 : a.token;
    *logp = none ? -INFINITY : -logf(a.s);
}
// the smallest of the lanes' numbers, in all of them
__device__ __forceinline__ int con_wave_min(int v) {
#define CON_DPP_MIN(ctrl, rows)                                                          \
    {                                                                                    \
        const int o = __builtin_amdgcn_update_dpp(v, v, (ctrl), (rows), 0xf, false);     \
        v = o < v ? o : v;                                                               \
    }
    CON_DPP_MIN(0x111, 0xf) CON_DPP_MIN(0x112, 0xf) CON_DPP_MIN(0x114, 0xf) CON_DPP_MIN(0x118, 0xf)  // row_shr 1, 2, 4, 8
    CON_DPP_MIN(0x142, 0xa) CON_DPP_MIN(0x143, 0xc)                                                  // row_bcast 15, 31
#undef CON_DPP_MIN
    return __builtin_amdgcn_readlane(v, 63);
}

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

template <typename T, int NT, int NV, bool PICK>
__global__ __launch_bounds__(NT) void constrain_kernel(const T* x, long ldx, T* y /* may be x */, long ldy, int V, int nseg, int per,
                                                        saConstraints C, PickPart* __restrict__ part, long long* __restrict__ tokens,
                                                        float* __restrict__ logp) {
    constexpr int VEC = SaVec<T>::N, SEG = NT * NV * VEC;
    extern __shared__ uint4 words4[];  // SEG words, then a position (16 bits) an entry, SEG at most; nothing where there are no lists
    __shared__ int found;
    __shared__ PickPart waves[NT / 64];
    unsigned* const words = (unsigned*)words4;
    const int row = blockIdx.x / nseg, seg = blockIdx.x % nseg, tid = threadIdx.x;
    const T* xr = x + (long)row * ldx;
    const int first = seg * per * VEC - sa_lead(xr), end = first + per * VEC < V ? first + per * VEC : V;
    // Everything the row needs from memory is asked for at once, the lists first: their atomics are the longer way.
    const bool lists = C.history || C.bias_ids;
    constexpr int AHEAD = 8;  // history entries a thread has in flight
    long long past[AHEAD], biased = -1;
    const long long* h = C.history + (long)row * C.history_ld;
    const long long* ids = C.bias_ids + (long)row * C.bias_ld;
    if (C.history)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) past[u] = u * NT + tid < C.history_len ? h[u * NT + tid] : -1;
    if (C.bias_ids && tid < C.n_bias) biased = ids[tid];
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = sa_load_vec(xr, first + (i * NT + tid) * VEC, end);
    const unsigned* mask = nullptr;
    if (C.mask) {
        const int state = C.states ? C.states[row] : row;
        if (state >= 0 && state < C.n_states) mask = C.mask + (long)state * C.mask_ld;
    }
    unsigned allowed[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v0 = first + (i * NT + tid) * VEC;
        allowed[i] = mask && v0 < end ? con_allowed<VEC>(mask, v0, V) : ~0u;
    }
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
#pragma unroll
        for (int i = 0; i < SEG / 4 / NT; ++i) words4[i * NT + tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) found = 0;
        // (a token t of a list is the segment's when `first` <= t < `end`; t >= 0 keeps what lies before the row out; the last
        // segment of a row that starts on a boundary may be empty, and begin behind the row's end)
        const unsigned long long n = end > first ? (unsigned long long)(end - first) : 0ull;
        auto add_bias = [&](long long t, int j) {
            const unsigned long long d = (unsigned long long)(t - first);
            if (t >= 0 && d < n && atomicMax(&words[d], (unsigned)(j + 1) << 16) == 0) places[atomicAdd(&found, 1)] = (sa_u16)d;
        };
        auto add_past = [&](long long t) {
            const unsigned long long d = (unsigned long long)(t - first);
            if (t >= 0 && d < n && atomicAdd(&words[d], 1u) == 0) places[atomicAdd(&found, 1)] = (sa_u16)d;
        };
        __syncthreads();
        if (C.bias_ids) {
            if (tid < C.n_bias) add_bias(biased, tid);
            for (int j = NT + tid; j < C.n_bias; j += NT) add_bias(ids[j], j);
            __syncthreads();
        }
        if (len > 0) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (u * NT + tid < len) add_past(past[u]);
            for (int i = AHEAD * NT; i < len; i += AHEAD * NT) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) past[u] = i + u * NT + tid < len ? h[i + u * NT + tid] : -1;
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) add_past(past[u]);
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
    float val[PICK ? NV * VEC : VEC], top = -INFINITY;
    int token = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int q = i * NT + tid, v0 = first + q * VEC;
        float* g = val + (PICK ? i * VEC : 0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = sa_element<T>(raw[i], e);
        if (lists) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const uint4 w = words4[(q * VEC + e) / 4];
                g[e] = w.x ? __builtin_bit_cast(float, w.x) : g[e];
                g[e + 1] = w.y ? __builtin_bit_cast(float, w.y) : g[e + 1];
                g[e + 2] = w.z ? __builtin_bit_cast(float, w.z) : g[e + 2];
                g[e + 3] = w.w ? __builtin_bit_cast(float, w.w) : g[e + 3];
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[e] = (allowed[i] >> e) & 1u ? g[e] : -INFINITY;
        if constexpr (PICK) {  // (what lies outside the row was loaded as -inf and is in no list)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (g[e] > top) { top = g[e]; token = v0 + e; }
        } else if (v0 < end) {
            sa_store_vec<T>(yr, v0, end, g, aligned);
        }
    }
    if constexpr (PICK) {
        const int lane = tid & 63;
        const float m = sa_wave_max_dpp(top), b = m > -INFINITY ? m : 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV * VEC; ++i) s += con_exp(val[i], b);
        s = sa_wave_sum_dpp(s);
        PickPart p{sa_order(m), con_wave_min(top == m ? token : 0x7fffffff), m, s};
        if (s != s) {  // a NaN: the first one is the largest value
            token = 0x7fffffff;
#pragma unroll
            for (int i = NV - 1; i >= 0; --i)
#pragma unroll
                for (int e = VEC - 1; e >= 0; --e)
                    if (val[i * VEC + e] != val[i * VEC + e]) token = first + (i * NT + tid) * VEC + e;
            p.best = sa_order(NAN);
            p.token = con_wave_min(token);
        }
        if (lane == 0) waves[tid >> 6] = p;
        __syncthreads();
        if (tid == 0) {
            PickPart r = waves[0];
#pragma unroll
            for (int w = 1; w < NT / 64; ++w) {
                pick_better(r, waves[w].best, waves[w].token);
                r.m = fmaxf(r.m, waves[w].m);
            }
            r.s = 0.0f;
#pragma unroll
            for (int w = 0; w < NT / 64; ++w)
                if (waves[w].s != 0.0f) r.s += waves[w].s * con_exp(waves[w].m, r.m);
            if (nseg == 1) pick_write(r, tokens + row, logp + row);
            else part[blockIdx.x] = r;
        }
    }
}

// the segments of a row, by one wave
__global__ __launch_bounds__(64) void pick_join_kernel(const PickPart* __restrict__ part, int nseg, long long* __restrict__ tokens,
                                                       float* __restrict__ logp) {
    const PickPart* P = part + (long)blockIdx.x * nseg;
    PickPart r{0u, 0x7fffffff, -INFINITY, 0.0f};
    for (int i = threadIdx.x; i < nseg; i += 64) {
        const PickPart p = P[i];
        pick_better(r, p.best, p.token);
        const float m = fmaxf(r.m, p.m);
        r.s = (r.s != 0.0f ? r.s * con_exp(r.m, m) : 0.0f) + (p.s != 0.0f ? p.s * con_exp(p.m, m) : 0.0f);
        r.m = m;
    }
    const float m = sa_wave_max_dpp(r.m);
    r.s = sa_wave_sum_dpp(r.s != 0.0f ? r.s * con_exp(r.m, m) : 0.0f);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) pick_better(r, (unsigned)__shfl_xor((int)r.best, o, 64), __shfl_xor(r.token, o, 64));
    if (threadIdx.x == 0) pick_write(r, tokens + blockIdx.x, logp + blockIdx.x);
}

// Threads, vectors a thread, segments a row, vectors a segment.  Segments of 4096 tokens -- each reads the lists of its row again,
// and three times as many of them run on a CU as of 8192 by the same 256 threads (256 x 131072 f32, history 4096: 71 us; 8192 tokens
// 85, 2048 tokens 82) -- and shorter ones where that leaves CUs without work.  Long lists are worth 512 threads and 8192 tokens, half
// as many looks at the lists by as many waves (61 -> 52 us with everything in the caches, history 1500 45 -> 44, 65535 365 -> 253;
// 1024 threads 56, 45, 236), where three of those workgroups come to every CU.  Where it saves pick its second launch, one workgroup
// takes a row of up to 8192.
struct ConPlan { int nt, nv, nseg, per; };
ConPlan con_plan(int rows, int V, int dtype, bool pick, int entries) {
    const int vec = dtype == SA_F32 ? 4 : 8, most = 16 / vec, vectors = (V + 2 * vec - 2) / vec;
    ConPlan p{256, 1, 1, 0};
    const bool whole = pick && vectors <= 512 * most;
    while (256 * p.nv < vectors &&
           (whole || (p.nv < most && (long)rows * ((vectors + 512 * p.nv - 1) / (512 * p.nv)) >= 512)))
        p.nv *= 2;
    if (!pick && entries > 1024 && vectors > 256 * most && (long)rows * ((vectors + 512 * most - 1) / (512 * most)) >= 768) p.nt = 512;
    p.nseg = (vectors + p.nt * p.nv - 1) / (p.nt * p.nv);
    p.per = (vectors + p.nseg - 1) / p.nseg;
    p.nseg = (vectors + p.per - 1) / p.per;
    return p;
}

bool con_ok(const saConstraints* c, int rows, int V) {
    if (!c || c->history_len < 0 || c->history_len > SA_LIST_MAX || c->n_bias < 0 || c->n_bias > SA_LIST_MAX) return false;
    // (without a request nothing is read: an empty list has no address)
    if (c->history_len > 0 && ((rows > 0 && !c->history) || c->history_ld < 0)) return false;
    if (c->n_bias > 0 && ((rows > 0 && (!c->bias_ids || !c->bias_values)) || c->bias_ld < 0)) return false;
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
    const dim3 grid((unsigned)((size_t)rows * p.nseg)), block(p.nt);
    const size_t segment = (size_t)p.nt * p.nv * SaVec<T>::N, entries = (size_t)c.history_len + c.n_bias;
    const size_t smem = entries ? segment * 4 + (entries < segment ? entries : segment) * 2 : 0;
#define CON_LAUNCH(NT, NV)                                                                                                        \
    hipLaunchKernelGGL((constrain_kernel<T, NT, NV, PICK>), grid, block, smem, stream, (const T*)x, ldx, (T*)y, ldy, V, p.nseg, p.per, \
                       C, part, tokens, logp)
    if (p.nt == 512) {
        if constexpr (!PICK) CON_LAUNCH(512, 16 / SaVec<T>::N);
    } else if (p.nv == 1) CON_LAUNCH(256, 1);
    else if (p.nv == 2) CON_LAUNCH(256, 2);
    else if constexpr (PICK || sizeof(T) == 4) {  // (con_plan's most: 16 / VEC, twice that for pick)
        if (p.nv == 4) CON_LAUNCH(256, 4);
        else if constexpr (PICK && sizeof(T) == 4) CON_LAUNCH(256, 8);
    }
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
    const ConPlan p = con_plan(rows, V, dtype, false, c->history_len + c->n_bias);
    if (!x || !y || !sa_threads_ok((long)rows * p.nseg, p.nt)) return CTC_STATUS_INVALID_VALUE;
    con_run<false>(x, ldx, dtype, y, ldy, rows, V, p, *c, nullptr, nullptr, nullptr, (hipStream_t)stream);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}

extern "C" size_t sa_logits_pick_workspace_bytes(int rows, int V, int dtype) {
    if (rows < 1 || !sa_rows_ok(dtype, V)) return 0;
    const ConPlan p = con_plan(rows, V, dtype, true, 0);
    return p.nseg == 1 ? 0 : (size_t)rows * p.nseg * sizeof(PickPart);
}

extern "C" ctcStatus_t sa_logits_pick(const void* x, long ldx, int dtype, int rows, int V, const saConstraints* c,
                                      long long* d_tokens, float* d_logp, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    SA_CLEAR_ERR();
    if (rows < 0 || !sa_rows_ok(dtype, V) || !con_ok(c, rows, V)) return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const ConPlan p = con_plan(rows, V, dtype, true, 0);
    const size_t need = sa_logits_pick_workspace_bytes(rows, V, dtype);
    if (!x || !d_tokens || !d_logp || (need && (!workspace || workspace_bytes < need)) || !sa_threads_ok((long)rows * p.nseg, 256))
        return CTC_STATUS_INVALID_VALUE;
    con_run<true>(x, ldx, dtype, nullptr, 0, rows, V, p, *c, (PickPart*)workspace, d_tokens, d_logp, (hipStream_t)stream);
    if (need)
        hipLaunchKernelGGL(pick_join_kernel, dim3(rows), dim3(64), 0, (hipStream_t)stream, (const PickPart*)workspace, p.nseg,
                           d_tokens, d_logp);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
