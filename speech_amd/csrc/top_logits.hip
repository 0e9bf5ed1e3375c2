// top_logits.hip -- the k largest logits of every row and the log-sum-exp of the others (sa_top_logits): what a teacher's row
// leaves for a distillation loss.
//
// Values are ordered as (value, lower index first) packed into one 64-bit number (sa_rank_key): all keys of a row differ, so the
// k-th is one element and ties go to the lowest index whatever the order of the work.
//
// One pass over the data.  A workgroup holds a segment of a row in registers.  The k-th largest of its threads' maxima is a bound
// that at least k elements reach and that only k threads' elements can pass: what reaches it are the candidates, a little more
// than k of thousands in ordinary rows, and everything below it goes straight into the log-sum-exp, relative to the bound.  The
// candidates are ranked against each other in LDS.  Where that does not hold -- rows that are masked or constant but for a few
// elements, NaN, a rest that vanishes beside the bound -- the workgroup looks for a better cut by halving, at a pass over the row in
// the caches for each step (4096 x 32000 bf16, k = 64, constant rows: 240 us a call against 80 for ordinary ones).
#include "rows.h"

namespace {

constexpr int kCand = 256;  // candidates a workgroup can hold: k <= 128 of them are kept

struct TopOut {
    float* values;
    long long* ids;
    float* rest;
};

// what a segment leaves for its row, beside `cap` candidates (0: none)
struct TopPart {
    float m, s;  // the others: maximum (or any bound close above it) and the sum of exp((x - m) / T); s = 0: none
};

__device__ __forceinline__ float top_exp(float x, float m, float c) { return x == m ? 1.0f : sa_exp2((x - m) * c); }

// The maximum over 1, 2 or 4 neighbouring lanes, in all of them: 256 keys a workgroup whatever its size
template <int LANES> __device__ __forceinline__ unsigned top_group(unsigned v) {
    if (LANES >= 2) {
        const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false);  // quad_perm 1,0,3,2
        v = o > v ? o : v;
    }
    if (LANES >= 4) {
        const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false);  // quad_perm 2,3,0,1
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ unsigned top_wave_max(unsigned v) {  // row_shr 1, 2, 4, 8, row_bcast 15, 31
#define TOP_DPP_MAX(ctrl, rows)                                                                          \
    {                                                                                                    \
        const unsigned o = (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, (ctrl), (rows), 0xf, false); \
        v = o > v ? o : v;                                                                               \
    }
    TOP_DPP_MAX(0x111, 0xf) TOP_DPP_MAX(0x112, 0xf) TOP_DPP_MAX(0x114, 0xf) TOP_DPP_MAX(0x118, 0xf)
    TOP_DPP_MAX(0x142, 0xa) TOP_DPP_MAX(0x143, 0xc)
#undef TOP_DPP_MAX
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// A number that at least k of this wave's 64 * N keys reach, and few more than k: halving the stretch between the smallest and the
// largest key until few enough do or the k-th key itself is found.  The low `shift` bits of the keys say nothing (logits of two
// bytes) and are not searched.  Uniform over the wave.
template <int N> __device__ __forceinline__ unsigned top_bound(unsigned (&key)[N], int k, int shift) {
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] >>= shift;
    unsigned hi = key[0], lo = key[0];
#pragma unroll
    for (int i = 1; i < N; ++i) {
        hi = key[i] > hi ? key[i] : hi;
        lo = key[i] < lo ? key[i] : lo;
    }
    hi = top_wave_max(hi) + 1u;  // (no key is all ones: sa_order)
    lo = ~top_wave_max(~lo);
    while (hi - lo > 1) {  // at least k keys reach lo, fewer reach hi
        const unsigned u = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(key[i] >= u));
        if (c < k) { hi = u; continue; }
        lo = u;
        if (c <= k + (k >> 3)) break;
    }
    return lo << shift;
}

// the low bits of a key, which no logit of the type sets differently from its sign
template <typename T> struct TopShift { static constexpr int value = 0; };
template <> struct TopShift<SaBf16> { static constexpr int value = 16; };
template <> struct TopShift<SaF16> { static constexpr int value = 13; };

// the lowest order of a logit that reaches `bound`: below zero the bits that say nothing are all ones
__device__ __forceinline__ unsigned top_low(unsigned bound, int shift) { return bound >> 31 ? bound : bound | ((1u << shift) - 1u); }

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
// (the candidates themselves lie in the order of their arrival, which no result may depend on) and returns the k-th key.  All
// threads count: 128 candidates at a time, NT / 128 stretches of the list each.
struct TopRank {
    unsigned long long cand[kCand], kth;
    int rank[kCand];
    float others[kCand];
};
template <int NT>
__device__ __forceinline__ unsigned long long top_rank(TopRank& R, int C, int k, long row, const TopOut& out) {
    constexpr int WIDE = NT < 128 ? NT : 128, PARTS = NT / WIDE;
    const int tid = threadIdx.x, part = tid / WIDE;
    for (int c = tid; c < kCand; c += NT) R.rank[c] = 0;
    const int each = (C + PARTS - 1) / PARTS, from = part * each, to = from + each < C ? from + each : C;
    __syncthreads();
    for (int c = tid % WIDE; c < C; c += WIDE) {
        const unsigned long long key = R.cand[c];
        int rank = 0;
#pragma unroll 4
        for (int j = from; j < to; ++j) rank += R.cand[j] > key;
        if (rank) atomicAdd(&R.rank[c], rank);
    }
    __syncthreads();
    for (int c = tid; c < C; c += NT) {
        const unsigned long long key = R.cand[c];
        const int rank = R.rank[c];
        const float f = sa_unorder((unsigned)(key >> 32));
        if (rank < k) {
            out.values[row * k + rank] = f;
            out.ids[row * k + rank] = (long long)(unsigned)~(unsigned)key;
            if (rank == k - 1) R.kth = key;
        } else {
            R.others[rank - k] = f;
        }
    }
    __syncthreads();
    return R.kth;
}

__device__ __forceinline__ void top_write_rest(float m, float s, float temperature, float* rest) {
    *rest = s == 0.0f ? -INFINITY : m / temperature + logf(s);
}

// A segment of a row: `per` <= NT * NV vectors; nseg == 1: the whole row, and the result.  (The segments of a row are of equal
// length: a short last one would have fewer than k threads with anything, no bound, and take the exact way.)
// It is a chain of short phases, and what hides one is another workgroup's: registers for six waves a SIMD (4096 x 32000 bf16, k = 64:
// 80 us a call, 82 - 88 a launch under the profiler, where the bytes alone would take 52).  Compared in runs that put it at 81:
// registers for eight waves, with spills, 128; unbounded 132; without the exponentials 75, without the ranking 76, with a bound known
// beforehand 58: no one phase bounds it.
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(6))) void top_segment_kernel(
    const T* __restrict__ x, SaRows at, int V, int k, int cap, float temperature, int nseg, int per, TopOut out,
    unsigned long long* __restrict__ lists, TopPart* __restrict__ parts) {
    constexpr int VEC = SaVec<T>::N;
    __shared__ TopRank R;
    // one key a thread, or, in rows so short that k threads might not have one, a key an element
    constexpr int KEYS = NT == 64 ? 64 : NV == 1 ? NT * VEC : 256;
    __shared__ unsigned top[KEYS], bound;
    __shared__ int count, counts[NT / 64];
    __shared__ float sums[NT / 64];
    const long row = blockIdx.x / nseg;
    const int seg = blockIdx.x % nseg, tid = threadIdx.x;
    const T* xr = x + at.at(row);
    const int first = seg * per * VEC - sa_lead(xr);  // the segment's first element (may lie before the row)
    const int end = first + per * VEC < V ? first + per * VEC : V;
    const float c = SA_LOG2E / temperature;
    constexpr bool TIGHT = NV * VEC > 32;
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = sa_load_vec<T, TIGHT>(xr, first + (i * NT + tid) * VEC, end);
    const int lo = first < 0 ? 0 : first, valid = end > lo ? end - lo : 0;

    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) mx = fmaxf(mx, sa_element<T>(raw[i], e));
    // (two-byte logits are widened again for every use: kept as 32 bits over the barriers they would take twice the registers)
    auto again = [&] {
        if constexpr (sizeof(T) == 2)
#pragma unroll
            for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
    };
    again();
    if constexpr (NT == 64) {  // one wave: eight keys a lane, and no exchange
        constexpr int GROUP = NV * VEC / 8;
        unsigned key[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            float m = -INFINITY;
#pragma unroll
            for (int j = g * GROUP; j < (g + 1) * GROUP; ++j) m = fmaxf(m, sa_element<T>(raw[j / VEC], j % VEC));
            key[g] = sa_order(m);
        }
        const unsigned t = top_bound(key, k, TopShift<T>::value);
        if (tid == 0) { bound = t; count = 0; }
    } else {
        if constexpr (NV == 1) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float f = sa_element<T>(raw[0], e);
                top[e * NT + tid] = f == f ? sa_order(f) : 0u;
            }
        } else {
            const unsigned u = top_group<(NT < 256 ? 256 : NT) / 256>(sa_order(mx));
            if (tid % ((NT + 255) / 256) == 0) top[tid / ((NT + 255) / 256)] = u;
        }
        if (tid == 0) count = 0;
        __syncthreads();
        if (tid < 64) {
            unsigned key[KEYS / 64];
#pragma unroll
            for (int i = 0; i < KEYS / 64; ++i) key[i] = top[tid + 64 * i];
            const unsigned t = top_bound(key, k, TopShift<T>::value);
            if (tid == 0) bound = t;
        }
    }
    __syncthreads();
    const float b = bound <= sa_order(-INFINITY) ? -INFINITY : sa_unorder(bound);
    // The others' sum, relative to the bound, and a bit for every element that reaches it.  (One multiply-add an element: the rounding
    // of b c is a common factor of all terms, no more than the bound's own last place in the logarithm.)
    constexpr int EACH = NV * VEC, WORDS = (EACH + 31) / 32, BITS = EACH < 32 ? EACH : 32;
    const float bc = b * c;
    unsigned hits[WORDS] = {};
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float f = sa_element<T>(raw[i], e), u = sa_exp2(__builtin_fmaf(f, c, -bc));
            const bool hit = f >= b;
            s += hit ? 0.0f : u;  // (NaN stays in the sum)
            hits[(i * VEC + e) / 32] = hits[(i * VEC + e) / 32] * 2u + (hit ? 1u : 0u);
            if (e == VEC - 1) __builtin_amdgcn_sched_barrier(0);  // (one vector after the other: fewer registers, 85 -> 81 us)
        }
    // Most threads that have one have one: their maximum.  The others' are read again (they were here a moment ago), two at a time.
    unsigned long long left = 0;  // the first element in the highest bit
#pragma unroll
    for (int w = 0; w < WORDS; ++w) left |= (unsigned long long)hits[w] << (64 - BITS * (w + 1));
    const int n = __popcll(left);
    if (n) {
        auto place = [&](int j) { return first + (j / VEC * NT + tid) * VEC + j % VEC; };
        auto add = [&](int v, float f) {
            if (v < 0 || v >= end) return true;  // (what the row does not have was loaded as -inf)
            const int p = atomicAdd(&count, 1);
            if (p < kCand) R.cand[p] = sa_rank_key(f, v);
            return p < kCand;
        };
        if (n == 1) {
            add(place(__builtin_clzll(left)), mx);
        } else {
            while (left) {
                const int j0 = __builtin_clzll(left), j1 = 63 - __builtin_ctzll(left), v0 = place(j0), v1 = place(j1);
                const float f0 = v0 >= 0 && v0 < end ? sa_widen(xr[v0]) : 0.0f, f1 = v1 >= 0 && v1 < end ? sa_widen(xr[v1]) : 0.0f;
                left &= ~(0x8000000000000000ull >> j0);
                bool room = add(v0, f0);
                if (j1 != j0) {
                    left &= ~(0x8000000000000000ull >> j1);
                    room = add(v1, f1);
                }
                if (!room && left) {  // too many: what is left is only counted
                    atomicAdd(&count, __popcll(left));
                    left = 0;
                }
            }
        }
    }
    s = sa_block_sum<NT / 64>(s, sums);
    if constexpr (NT == 64) __syncthreads();  // (one wave sums without a barrier)
    int C = count;
    float m = b;
    if (C > cap || (C < valid && !(s >= 0x1p-70f && s <= 2.0f * valid))) {
        // The row again, now with a cut that between min(k, valid) and `cap` elements reach: halving above the bound, then, where one
        // value alone has too many, over the index.  Each look at the row is a pass over what the caches hold of it.
        auto look = [&](int until, auto&& visit) __attribute__((always_inline)) {  // the elements below `until` <= end
#pragma unroll 2
            for (int i = 0; i < NV; ++i) {
                const int v0 = first + (i * NT + tid) * VEC;
                if (v0 >= until) break;
                const uint4 r = sa_load_vec<T, TIGHT>(xr, v0, end);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (v0 + e >= lo && v0 + e < until) visit(sa_element<T>(r, e), v0 + e);
            }
        };
        auto number = [](unsigned u) { return u > sa_order(INFINITY) ? NAN : sa_unorder(u); };  // (NaN: nothing but NaN reaches it)
        auto reaches = [&](float t) __attribute__((always_inline)) {
            int n = 0;
            look(end, [&](float f, int) { n += f >= t || f != f; });
            return top_count<NT>(n, counts);
        };
        const int want = k < valid ? k : valid;
        unsigned K = b == -INFINITY ? sa_order(-INFINITY) : top_low(bound, TopShift<T>::value);
        int places = end;  // of the elements equal to the cut, those below this index
        if (s != s) C = reaches(number(K));  // (a NaN reaches every cut)
        if (C > cap) {
            unsigned hi = 0xffffffffu, u = K + 1u;  // (the next value first: ties at the bound are the common case)
            int above = 0;                          // how many reach `hi`
            while (C > cap && hi - K > 1) {
                const int n = reaches(number(u));
                if (n >= want) { K = u; C = n; }
                else { hi = u; above = n; }
                u = K + (hi - K) / 2;
            }
            if (C > cap) {
                const float t = number(K);
                // fewer than `want` with the equal ones below `from`, more than `cap` with those below `places`: in between by the
                // share that is wanted, and every other time by half
                int from = lo, few = above;
                for (bool half = false; C > cap; half = !half) {
                    const long share = (long)(places - from) * ((want + cap) / 2 - few) / (C - few);
                    const int v = half || share < 1 ? from + (places - from) / 2 : from + (int)share;
                    int n = 0;
                    look(v, [&](float f, int) { n += f == t || (f != f && t != t); });
                    n = above + top_count<NT>(n, counts);
                    if (n < want) { from = v; few = n; }
                    else { places = v; C = n; }
                }
            }
        }
        const float t = number(K);
        auto taken = [&](float f, int v) __attribute__((always_inline)) { return f > t || (f != f && t == t) || ((f == t || (f != f && t != t)) && v < places); };
        __syncthreads();  // (nobody still has to read the first count: where it fits, no look at the row came in between)
        if (tid == 0) count = 0;
        __syncthreads();
        float most = -INFINITY;
        m = t;  // (the others' sum relative to the cut, unless they vanish beside it)
        s = 0.0f;
        look(end, [&](float f, int v) {
            if (taken(f, v)) {
                R.cand[atomicAdd(&count, 1)] = sa_rank_key(f, v);
            } else {
                s += top_exp(f, m, c);
                most = fmaxf(most, f);
            }
        });
        s = sa_block_sum<NT / 64>(s, sums);
        if (!(s >= 0x1p-70f) && C < valid) {
            m = sa_block_max<NT / 64>(most, sums);
            s = 0.0f;
            look(end, [&](float f, int v) { s += taken(f, v) ? 0.0f : top_exp(f, m, c); });
            s = sa_block_sum<NT / 64>(s, sums);
        }
    } else if (C == valid) {
        s = 0.0f;
    }
    if (s == 0.0f) m = -INFINITY;

    if (nseg > 1) {
        if (tid == 0) parts[blockIdx.x] = TopPart{m, s};
        __syncthreads();
        for (int i = tid; i < cap; i += NT) lists[(size_t)blockIdx.x * cap + i] = i < C ? R.cand[i] : 0;
        return;
    }
    top_rank<NT>(R, C, k, row, out);
    // the candidates that were not taken belong to the others
    const float mu = C > k ? R.others[0] : -INFINITY;
    float su = tid < C - k ? top_exp(R.others[tid], mu, c) : 0.0f;
    if constexpr (NT < kCand)
        for (int i = tid + NT; i < C - k; i += NT) su += top_exp(R.others[i], mu, c);
    su = sa_block_sum<NT / 64>(su, sums);
    if (tid == 0) {
        const float M = fmaxf(m, mu);
        top_write_rest(M, s * top_exp(m, M, c) + su * top_exp(mu, M, c), temperature, out.rest + row);
    }
}

// The segments of a row: the same over their candidates, nseg * cap <= NT * EACH keys, in registers.
template <int NT, int EACH>
__global__ __launch_bounds__(NT) void top_merge_kernel(const unsigned long long* __restrict__ lists, const TopPart* __restrict__ parts,
                                                       int nseg, int cap, int k, int shift, float temperature, TopOut out) {
    __shared__ TopRank R;
    __shared__ unsigned top[256], bound;
    __shared__ int count, counts[NT / 64];
    __shared__ float sums[NT / 64];
    __shared__ unsigned long long total;
    __shared__ int odd;
    const long row = blockIdx.x;
    const int tid = threadIdx.x, n = nseg * cap;
    const float c = SA_LOG2E / temperature;
    lists += (size_t)row * n;
    parts += (size_t)row * nseg;
    unsigned long long keys[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) keys[i] = i * NT + tid < n ? lists[i * NT + tid] : 0;
    const TopPart P = tid < nseg ? parts[tid] : TopPart{-INFINITY, 0.0f};  // (nseg <= 62 here with 256 threads, <= 257 with 1024)
    unsigned long long mx = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) mx = keys[i] > mx ? keys[i] : mx;
    const unsigned u = top_group<NT / 256>((unsigned)(mx >> 32));
    if (tid % (NT / 256) == 0) top[tid / (NT / 256)] = u;
    if (tid == 0) { count = 0; total = 0; odd = 0; }
    __syncthreads();
    if (tid < 64) {
        unsigned key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) key[i] = top[tid + 64 * i];
        const unsigned t = top_bound(key, k, shift);
        if (tid == 0) bound = t;
    }
    __syncthreads();
    const unsigned b = top_low(bound, shift);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (keys[i] && (unsigned)(keys[i] >> 32) >= b) {
            const int p = atomicAdd(&count, 1);
            if (p < kCand) R.cand[p] = keys[i];
        }
    __syncthreads();
    int C = count;
    if (C > kCand) {
        // halving until few enough reach K (all keys differ); the next value first: ties are the common case
        unsigned long long K = (unsigned long long)b << 32, hi = ~0ull, u = K + (1ull << 32);
        if (u < K) u = K + (hi - K) / 2;
        while (C > kCand) {
            int r = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i) r += keys[i] >= u;
            r = top_count<NT>(r, counts);
            if (r >= k) { K = u; C = r; }
            else hi = u;
            u = K + (hi - K) / 2;
        }
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (keys[i] >= K) R.cand[atomicAdd(&count, 1)] = keys[i];
    }
    const unsigned long long last = top_rank<NT>(R, C, k, row, out);
    // The others: the candidates that were not taken, and the segments' sums.  The reference is the largest TERM, not the largest
    // bound: a segment's sum may be as small as 2^-70 of its bound.
    float m = P.s != 0.0f ? P.m + sa_log2(P.s) / c : -INFINITY;
    unsigned long long left = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) left = keys[i] < last && keys[i] > left ? keys[i] : left;
    if (left) m = fmaxf(m, sa_unorder((unsigned)(left >> 32)));
    m = sa_block_max<NT / 64>(m, sums);
    float s = sa_block_sum<NT / 64>(P.s != 0.0f ? P.s * top_exp(P.m, m, c) : 0.0f, sums);
    // The lists are in the order of arrival: their terms (0 .. 1) are rounded to multiples of 2^-48 and summed as integers, the same in
    // any order.  28896 terms at most: the sum stays below 2^63, and all roundings together below 2^-34 of a sum of 1 or more.
    unsigned long long sum = 0;
    if (left) {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (keys[i] && keys[i] < last) {
                const float e = top_exp(sa_unorder((unsigned)(keys[i] >> 32)), m, c);
                if (e == e) sum += __float2ull_rn(e * 0x1p48f);
                else odd = 1;
            }
    }
    if (sum) atomicAdd(&total, sum);
    __syncthreads();
    s += odd ? NAN : (float)total * 0x1p-48f;
    if (tid == 0) top_write_rest(m, s, temperature, out.rest + row);
}

// Short rows (V <= 128): LANES lanes each, EACH elements a lane, every element ranked against all others.
template <typename T, int LANES, int EACH>
__global__ __launch_bounds__(256) void top_short_kernel(const T* __restrict__ x, SaRows at, long rows, int V, int k,
                                                        float temperature, TopOut out) {
    constexpr int ROWS = 256 / LANES;
    __shared__ unsigned long long keys[ROWS][LANES * EACH];
    const int lane = threadIdx.x % LANES, w = threadIdx.x / LANES;
    const long row = (long)blockIdx.x * ROWS + w;
    if (row >= rows) return;  // (no barrier below: a wave's LDS accesses are in order)
    const T* xr = x + at.at(row);
    const float c = SA_LOG2E / temperature;
    float f[EACH];
    unsigned long long key[EACH];
    int rank[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int v = lane + LANES * i;
        f[i] = v < V ? sa_widen(xr[v]) : -INFINITY;
        key[i] = v < V ? sa_rank_key(f[i], v) : 0;
        keys[w][v] = key[i];
        rank[i] = 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int j = 0; j < V; ++j) {
        const unsigned long long o = keys[w][j];
#pragma unroll
        for (int i = 0; i < EACH; ++i) rank[i] += o > key[i];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int v = lane + LANES * i;
        if (v >= V) continue;
        if (rank[i] < k) {
            out.values[row * k + rank[i]] = f[i];
            out.ids[row * k + rank[i]] = v;
        } else {
            m = fmaxf(m, f[i]);
        }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, LANES));
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (lane + LANES * i < V && rank[i] >= k) s += top_exp(f[i], m, c);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, LANES);
    if (lane == 0) top_write_rest(m, s, temperature, out.rest + row);
}

// Rows that a workgroup's registers hold are not split when there are enough of them to fill the device (4096 x 32000 bf16, in the same
// runs: 81 us whole, 90 + 23 in two segments and a merge), and a wave takes a row of up to 1000 (2000 of two bytes) when every SIMD gets one:
// no exchange between waves (16000 x 1000 f32, k = 8: 25 us against 58 with 256 threads; 16000 x 1000 bf16, k = 64: 40 against 98; at twice
// the length 33 against 36 and 32 against 30).  Others are split into segments of 256 threads, shorter ones where there are few
// rows, as long as one workgroup can hold what the segments leave.
struct TopPlan {
    int nt, nv, nseg, per, cap;  // threads, vectors a thread, segments a row, vectors a segment, candidates a segment leaves
};
TopPlan top_plan(long rows, int V, int k, int dtype) {
    const int vec = dtype == SA_F32 ? 4 : 8, vectors = (V + vec - 1 + vec - 1) / vec;  // the longest row, with its lead
    TopPlan p{256, 8, 1, vectors, k + k / 2 + 32};
    if (vectors <= 64 * 4 && rows >= 1024) {
        p.nt = 64;
        p.nv = vectors <= 128 ? 2 : 4;
    } else if (vectors <= 256 * 8) {
        p.nv = vectors <= 256 ? 1 : vectors <= 512 ? 2 : vectors <= 1024 ? 4 : 8;
    } else if (vectors <= 1024 * 8 && rows >= 256) {
        p.nt = vectors <= 512 * 8 ? 512 : 1024;
    } else {
        if (rows * ((vectors + 2047) / 2048) < 128 && (vectors + 1023) / 1024 * p.cap <= 16384) p.nv = 4;
        p.nseg = (vectors + 256 * p.nv - 1) / (256 * p.nv);
        p.per = (vectors + p.nseg - 1) / p.nseg;
        p.nseg = (vectors + p.per - 1) / p.per;
    }
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
#define TOP_SHORT(LANES, EACH)                                                                                             \
    hipLaunchKernelGGL((top_short_kernel<T, LANES, EACH>), dim3((unsigned)((rows * LANES + 255) / 256)), dim3(256), 0, stream, xt, \
                       at, rows, V, k, temperature, out)
        if (V <= 32) TOP_SHORT(32, 1);
        else if (V <= 64) TOP_SHORT(64, 1);
        else TOP_SHORT(64, 2);
#undef TOP_SHORT
        return;
    }
    TopPart* parts = (TopPart*)ws;
    unsigned long long* lists = (unsigned long long*)(ws + sa_align_up((size_t)rows * p.nseg * sizeof(TopPart), 256));
    const int cap = p.nseg == 1 ? kCand : p.cap, n = p.nseg * p.cap;
    const dim3 grid((unsigned)(rows * p.nseg)), block(p.nt);
#define TOP_LAUNCH(NT, NV)                                                                                                   \
    hipLaunchKernelGGL((top_segment_kernel<T, NT, NV>), grid, block, 0, stream, xt, at, V, k, cap, temperature, p.nseg, p.per, out, \
                       lists, parts)
    if (p.nt == 64 && p.nv == 2) TOP_LAUNCH(64, 2);
    else if (p.nt == 64) TOP_LAUNCH(64, 4);
    else if (p.nt == 1024) TOP_LAUNCH(1024, 8);
    else if (p.nt == 512) TOP_LAUNCH(512, 8);
    else if (p.nv == 1) TOP_LAUNCH(256, 1);
    else if (p.nv == 2) TOP_LAUNCH(256, 2);
    else if (p.nv == 4) TOP_LAUNCH(256, 4);
    else TOP_LAUNCH(256, 8);
#undef TOP_LAUNCH
    if (p.nseg == 1) return;
#define TOP_MERGE(NT, EACH)                                                                                            \
    hipLaunchKernelGGL((top_merge_kernel<NT, EACH>), dim3((unsigned)rows), dim3(NT), 0, stream, (const unsigned long long*)lists, \
                       (const TopPart*)parts, p.nseg, p.cap, k, TopShift<T>::value, temperature, out)
    if (n <= 256 * 8) TOP_MERGE(256, 8);
    else if (n <= 1024 * 8) TOP_MERGE(1024, 8);
    else TOP_MERGE(1024, 32);  // (129 segments of 224 at most: 28896 keys)
#undef TOP_MERGE
}

bool top_ok(long rows, int V, int k, int dtype) {
    if (rows < 0 || rows > 0x7fffffffL || !sa_rows_ok(dtype, V) || k < 1 || k > V || k > SA_TOP_MAX) return false;
    if (V <= 128) return sa_threads_ok(rows, V <= 32 ? 32 : 64);
    const TopPlan p = top_plan(rows, V, k, dtype);
    return sa_threads_ok(rows * p.nseg, p.nt) && (p.nseg == 1 || sa_threads_ok(rows, 1024));
}

}  // namespace

extern "C" size_t sa_top_logits_workspace_bytes(long rows, int V, int k, int dtype) {
    return top_ok(rows, V, k, dtype) ? top_bytes(rows, top_plan(rows, V, k, dtype)) : 0;
}

extern "C" ctcStatus_t sa_top_logits(const void* x, long ld_outer, long ld_inner, int n_inner, int dtype, long rows, int V,
                                     int k, float temperature, float* values, long long* ids, float* rest, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    SA_CLEAR_ERR();
    if (!top_ok(rows, V, k, dtype) || n_inner < 1 || !sa_temperature_ok(temperature))
        return CTC_STATUS_INVALID_VALUE;
    if (rows == 0) return CTC_STATUS_SUCCESS;
    const TopPlan p = top_plan(rows, V, k, dtype);
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
