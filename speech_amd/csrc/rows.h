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

static inline size_t sa_type_bytes(int dtype) { return dtype == SA_F32 ? 4 : 2; }
static inline bool sa_rows_ok(int dtype, int V) { return dtype >= SA_F32 && dtype <= SA_F16 && V >= 1 && V <= SA_VOCAB_MAX; }

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
