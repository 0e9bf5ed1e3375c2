// rows.h -- what the operators on output rows share (constrain.hip, top_logits.hip, distill.hip): the element types of the
// logits, where a row starts, and reductions over the waves of a block.  A row is the V logits of one token.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "internal.h"

typedef unsigned short sa_u16;
struct SaBf16 { sa_u16 v; };
struct SaF16 { sa_u16 v; };

__device__ __forceinline__ float sa_widen(float x) { return x; }
__device__ __forceinline__ float sa_widen(SaBf16 x) { return __builtin_bit_cast(float, (unsigned)x.v << 16); }
__device__ __forceinline__ float sa_widen(SaF16 x) { return (float)__builtin_bit_cast(_Float16, x.v); }
// the only rounding to the logits' type: to nearest even, once, of a result held in 32 bits
template <typename T> __device__ __forceinline__ T sa_narrow(float x);
template <> __device__ __forceinline__ float sa_narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ SaBf16 sa_narrow<SaBf16>(float x) { return SaBf16{(sa_u16)(sa_cvt_pk_bf16(x, x) & 0xffffu)}; }
template <> __device__ __forceinline__ SaF16 sa_narrow<SaF16>(float x) { return SaF16{__builtin_bit_cast(sa_u16, (_Float16)x)}; }

// Row r of a (outer, inner, V) view whose last stride is one; a matrix has n_inner = 1.
struct SaRows {
    long ld_outer, ld_inner;
    int n_inner;
    __host__ __device__ __forceinline__ long at(long r) const {
        return n_inner == 1 ? r * ld_outer : (r / n_inner) * ld_outer + (r % n_inner) * ld_inner;
    }
};

static inline bool sa_temperature_ok(float t) { return t >= 0.99e-6f && t <= 1.01e6f; }  // T^2 and x / T stay in 32 bits
static inline bool sa_rows_ok(int dtype, int V) { return dtype >= SA_F32 && dtype <= SA_F16 && V >= 1 && V <= SA_VOCAB_MAX; }
// a launch holds fewer than 2^32 threads (its last workgroup filled up)
static inline bool sa_threads_ok(long groups, long threads) { return groups <= (0xffffffffL - 1023) / threads; }

// Sum / maximum over the NW waves of a block, the same value in every thread; `scratch` holds NW floats.  The waves' results
// are joined in the order of the waves: the same bits on every run.
template <int NW> __device__ __forceinline__ float sa_block_sum(float v, float* scratch) {
    v = sa_wave_sum_dpp(v);
    if (NW == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += scratch[w];
    return s;
}
template <int NW> __device__ __forceinline__ float sa_block_max(float v, float* scratch) {
    v = sa_wave_max_dpp(v);
    if (NW == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = scratch[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, scratch[w]);
    return m;
}

// A float as an unsigned number of the same order: NaN above everything (and below all ones, which no key of sa_rank_key is),
// -0 equal to +0 (so ties go by the index alone).
__device__ __forceinline__ unsigned sa_order(float x) {
    if (x != x) return 0xfffffffeu;
    const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sa_unorder(unsigned k) {  // the inverse
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// (value, index) as one number: larger value first, then the lower index
__device__ __forceinline__ unsigned long long sa_rank_key(float x, int i) {
    return ((unsigned long long)sa_order(x) << 32) | (unsigned)~(unsigned)i;
}

// ---- a row as vectors of 16 bytes ------------------------------------------------------------------------------------------
// Rows start anywhere (odd V, views): vector q of a row covers its elements [q VEC - lead, q VEC - lead + VEC), where `lead` is how
// many elements the row starts behind a 16-byte boundary.  Every whole vector is then one aligned 16-byte access and only a row's
// first and last vector can be partial: those are accessed by elements of the row alone, so nothing outside it is touched.
template <typename T> struct SaVec { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T> __device__ __forceinline__ unsigned sa_fill_word();  // -inf in every element
template <> __device__ __forceinline__ unsigned sa_fill_word<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ unsigned sa_fill_word<SaBf16>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ unsigned sa_fill_word<SaF16>() { return 0xfc00fc00u; }

__device__ __forceinline__ unsigned sa_bits(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ unsigned sa_bits(SaBf16 x) { return x.v; }
__device__ __forceinline__ unsigned sa_bits(SaF16 x) { return x.v; }

template <typename T> __device__ __forceinline__ int sa_lead(const T* row) { return (int)(((uintptr_t)row & 15) / sizeof(T)); }

template <typename T> __device__ __forceinline__ float sa_element(const uint4& q, int e);
template <> __device__ __forceinline__ float sa_element<float>(const uint4& q, int e) {
    return __builtin_bit_cast(float, e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w);
}
template <> __device__ __forceinline__ float sa_element<SaBf16>(const uint4& q, int e) {
    const unsigned w = e < 2 ? q.x : e < 4 ? q.y : e < 6 ? q.z : q.w;
    return __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
}
template <> __device__ __forceinline__ float sa_element<SaF16>(const uint4& q, int e) {
    const unsigned w = e < 2 ? q.x : e < 4 ? q.y : e < 6 ? q.z : q.w;
    return (float)__builtin_bit_cast(_Float16, (sa_u16)(e & 1 ? w >> 16 : w));
}

// element e becomes -inf
template <typename T> __device__ __forceinline__ void sa_drop_element(uint4& q, int e) {
    constexpr int per = 4 / (int)sizeof(T);
    unsigned* const w[4] = {&q.x, &q.y, &q.z, &q.w};
    unsigned& u = *w[e / per];
    if constexpr (per == 1) u = sa_fill_word<T>();
    else u = e & 1 ? (u & 0xffffu) | (sa_fill_word<T>() & 0xffff0000u) : (u & 0xffff0000u) | (sa_fill_word<T>() & 0xffffu);
}

// eight or four results, rounded to the type
template <typename T> __device__ __forceinline__ uint4 sa_pack(const float* g);
template <> __device__ __forceinline__ uint4 sa_pack<float>(const float* g) {
    return make_uint4(__builtin_bit_cast(unsigned, g[0]), __builtin_bit_cast(unsigned, g[1]), __builtin_bit_cast(unsigned, g[2]),
                      __builtin_bit_cast(unsigned, g[3]));
}
template <> __device__ __forceinline__ uint4 sa_pack<SaBf16>(const float* g) {
    return make_uint4(sa_cvt_pk_bf16(g[0], g[1]), sa_cvt_pk_bf16(g[2], g[3]), sa_cvt_pk_bf16(g[4], g[5]), sa_cvt_pk_bf16(g[6], g[7]));
}
template <> __device__ __forceinline__ uint4 sa_pack<SaF16>(const float* g) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = (unsigned)sa_narrow<SaF16>(g[2 * i]).v | ((unsigned)sa_narrow<SaF16>(g[2 * i + 1]).v << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// the vector whose first element is v0, into a row that starts at the same offset from a 16-byte boundary
template <typename T> __device__ __forceinline__ void sa_store_vec(T* row, int v0, int V, const float* g, bool aligned) {
    if (aligned && v0 >= 0 && v0 + SaVec<T>::N <= V) {
        // (past the caches: what is written here is as large as what is read, and reads again come first; 2048 x 131072 f32 gradients
        // 470 -> 440 us)
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        const uint4 w = sa_pack<T>(g);
        __builtin_nontemporal_store((u4){w.x, w.y, w.z, w.w}, reinterpret_cast<u4*>(row + v0));
        return;
    }
#pragma unroll
    for (int e = 0; e < SaVec<T>::N; ++e)
        if (v0 + e >= 0 && v0 + e < V) row[v0 + e] = sa_narrow<T>(g[e]);
}

// The vector whose first element is v0 (a multiple of VEC minus lead); -inf outside [0, V).  A row's first and last vector: all their
// elements at once, those outside taken from the row's ends and dropped -- one wait, where one element after the other costs rows of
// odd lengths 10 - 20 % (8000 x 5001 bf16: top logits 48 -> 42 us, constrain 52 -> 43, distillation 54 -> 48).  The registers it takes
// cost rows without partial vectors something (pick, 4096 x 32000 bf16: 99 -> 108 us).  TIGHT: one after the other, for kernels that
// have none to spare (top logits, bf16: 83 us a launch against 86 at 4096 x 32000, but 94 against 86 at 4096 x 32001).
template <typename T, bool TIGHT = false> __device__ __forceinline__ uint4 sa_load_vec(const T* row, int v0, int V) {
    if (v0 >= 0 && v0 + SaVec<T>::N <= V) return *reinterpret_cast<const uint4*>(row + v0);
    constexpr int N = SaVec<T>::N, BITS = 8 * (int)sizeof(T);
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sa_fill_word<T>();
    if (v0 >= V) return make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (TIGHT) {
        unsigned long long u[2] = {(unsigned long long)w[1] << 32 | w[0], (unsigned long long)w[3] << 32 | w[2]};
#pragma unroll 1
        for (int e = 0; e < N; ++e) {
            const int v = v0 + e;
            if (v < 0 || v >= V) continue;
            const unsigned long long h = sa_bits(row[v]);
            const int at = e * BITS & 63;
            const unsigned long long keep = ~(((1ull << BITS) - 1) << at);
            if (e * BITS < 64) u[0] = (u[0] & keep) | h << at;
            else u[1] = (u[1] & keep) | h << at;
        }
        return make_uint4((unsigned)u[0], (unsigned)(u[0] >> 32), (unsigned)u[1], (unsigned)(u[1] >> 32));
    } else {
        unsigned h[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int v = v0 + e;
            h[e] = sa_bits(row[v < 0 ? 0 : v >= V ? V - 1 : v]);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int v = v0 + e;
            if constexpr (BITS == 32) {
                w[e] = v >= 0 && v < V ? h[e] : w[e];
            } else {
                const unsigned u = v >= 0 && v < V ? h[e] : sa_fill_word<T>() & 0xffffu;
                w[e / 2] = e & 1 ? w[e / 2] | u << 16 : u;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}
