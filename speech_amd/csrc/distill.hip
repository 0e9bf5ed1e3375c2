// distill.hip -- distillation from a teacher's top logits, loss and gradient (sa_distill_loss; the formulas are in
// include/speech_amd.h).
//
// exp2((x - m) log2 e / T) with the maximum subtracted FIRST: the difference of two close numbers is exact, and a row that is masked
// with the type's lowest value stays finite (a fused x c - m c would leave the rounding error of m c, which is huge there).
// The listed tokens and the rest have maxima and sums of their own: p_rest is a sum of its own terms and no difference from 1, and
// it does not vanish when the rest lies far below the list.
//
// A workgroup per row.  The row is read once, as 16-byte vectors, into registers (what is beyond NT * NV vectors is read a second
// time); each thread sums relative to its own maximum, the waves' results are joined in one exchange through LDS, and the
// gradient is formed from the registers: from the exponentials themselves where they fit (KEEP), one or two multiplications an
// element, else from the logits again.  At T = 2 and T = 4 the second sum takes exp(x - m) as a power of exp((x - m) / T): 4096 x 32000
// bf16 115 us a call where exponentials of its own, taken again for the gradient, cost 155, 2048 x 131072 f32 440 against 481, 1000 x
// 50021 f16 71 against 79; that is what other temperatures with hard targets cost (T = 3: 153, 480, 79).
// Listed tokens are marked in a bitmap in LDS and taken out of the sums where the rest is a class of its own; their gradients
// replace what the row-wide formula wrote.  The teacher's side of a row is k <= 128
// numbers: the first wave does it, two to a lane, while the others sum.
#include "rows.h"

namespace {

struct DisArgs {
    const float* values;
    const long long* ids;
    const float* rest;
    int k;
    const long long* targets;
    const float* weights;
    float temperature, alpha, scale;
    const float* factor;
    int skip_unit;
    float* loss_rows;
};

struct DisSum { float m, s, h; };  // maximum, sum of exp((x - m) / T), sum of exp(x - m)

// a maximum that can be subtracted: -inf (nothing there) counts as 0, and every exp2((-inf - 0) c) is 0
__device__ __forceinline__ float dis_base(float m) { return m == -INFINITY ? 0.0f : m; }

// REST: the rest is a class, and the list is taken out of the sums.  The sum at temperature 1 beside the one at T, HARD: 0 not wanted
// or the same; 1 by its own exponential; 2, 4 as that power of the one at T = 2, 4.
// MORE: rows longer than the registers hold.
template <typename T, int NT, int NV, bool MORE, bool REST, int HARD>
__global__ __launch_bounds__(NT) void distill_kernel(const T* __restrict__ x, T* dx, SaRows at, int V, int stash, DisArgs A) {
    constexpr int VEC = SaVec<T>::N, NW = NT / 64;
    constexpr bool TWO = HARD != 0, KEEP = HARD != 1;  // (only one exponential of an element is kept)
    extern __shared__ uint4 held[];                // `stash` vectors a thread, and behind them
    unsigned* bitmap = (unsigned*)(held + stash * NT);  // a bit per element of the row's vectors: the token is in the list
    __shared__ DisSum waves[NW];
    __shared__ int ids[SA_TOP_MAX];
    __shared__ float qs[SA_TOP_MAX];
    __shared__ float list[4];  // what the first wave found: maximum and sums over the list, q of the rest
    __shared__ int soft_row;
    const long row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    float f = A.scale;
    if (A.factor) {
        const float g = *A.factor;
        if (A.skip_unit && g == 1.0f) return;
        f *= g;
    }
    const float w = A.weights ? A.weights[row] : 1.0f;
    const T* xr = x + at.at(row);
    T* dr = dx ? dx + at.at(row) : nullptr;
    const int lead = sa_lead(xr);
    const bool aligned = dr && sa_lead(dr) == lead;
    const int nq = (V + lead + VEC - 1) / VEC;
    if (w == 0.0f) {  // nothing of the row is read: it may hold anything
        const float zero[VEC] = {};
        if (dr)
            for (int q = tid; q < nq; q += NT) sa_store_vec<T>(dr, q * VEC - lead, V, zero, aligned);
        if (A.loss_rows && tid == 0) A.loss_rows[row] = 0.0f;
        return;
    }
    f *= w;

    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = sa_load_vec(xr, (i * NT + tid) * VEC - lead, V);
    const long long target = A.alpha < 1.0f && A.targets ? A.targets[row] : -1;
    const bool hard = target >= 0 && target < V;
    const float xt = hard ? sa_widen(xr[target]) : 0.0f;
    // the list: marked in the bitmap by the first wave, two entries a lane
    int id[2] = {-1, -1};
    float a[2] = {-INFINITY, -INFINITY}, xv[2] = {-INFINITY, -INFINITY};
    for (int i = tid; i < (nq * VEC + 31) / 32; i += NT) bitmap[i] = 0;
    if (tid < 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = lane + 64 * i;
            if (j >= A.k) continue;
            const long long t = A.ids[row * A.k + j];
            if (t >= 0 && t < V) {
                id[i] = (int)t;
                a[i] = A.values[row * A.k + j] / A.temperature;
                xv[i] = sa_widen(xr[t]);
            }
        }
    }
    __syncthreads();
    bool twice = false;  // some id stands in the list more than once
    if (tid < 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = lane + 64 * i, p = id[i] + lead;
            if (id[i] >= 0) twice |= (atomicOr(&bitmap[p >> 5], 1u << (p & 31)) >> (p & 31)) & 1u;
            if (j < A.k) ids[j] = id[i];
        }
        twice = __any(twice);
    }
    __syncthreads();

    // the teacher: q of the list and of the rest; the student's sums over the list (each id once)
    const float c = SA_LOG2E / A.temperature;
    bool first[2] = {false, false}, soft = false;
    float q[2], qsum[2], am = 0.0f, lt = 0.0f, qr = 0.0f, ar = -INFINITY;
    if (tid < 64) {
        if (REST) ar = A.rest[row];
        am = fmaxf(sa_wave_max_dpp(fmaxf(a[0], a[1])), ar);
        // (a list that holds NaN, or +inf, has no distribution: q, the loss and the list's gradients become NaN, whatever else is there)
        soft = (am > -INFINITY || __any(a[0] != a[0] || a[1] != a[1] || ar != ar)) && A.alpha > 0.0f;
        const float e0 = soft ? sa_exp2((a[0] - am) * SA_LOG2E) : 0.0f, e1 = soft ? sa_exp2((a[1] - am) * SA_LOG2E) : 0.0f;
        const float er = soft && REST ? sa_exp2((ar - am) * SA_LOG2E) : 0.0f;
        const float total = sa_wave_sum_dpp(e0 + e1) + er;
        lt = logf(total);
        q[0] = soft ? e0 / total : 0.0f;
        q[1] = soft ? e1 / total : 0.0f;
        qr = soft ? er / total : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            first[i] = id[i] >= 0;
            qsum[i] = q[i];
            if (lane + 64 * i < A.k) qs[lane + 64 * i] = q[i];
        }
        if (twice) {  // in the order of the list, whoever marked the bit
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (id[i] < 0) continue;
                qsum[i] = 0.0f;
                for (int j = 0; j < A.k; ++j)
                    if (ids[j] == id[i]) {
                        if (j < lane + 64 * i) first[i] = false;
                        qsum[i] += qs[j];
                    }
            }
        }
        if (REST) {
            const float y0 = first[0] ? xv[0] : -INFINITY, y1 = first[1] ? xv[1] : -INFINITY;
            const float mt = sa_wave_max_dpp(fmaxf(y0, y1)), b = dis_base(mt);
            const float st = sa_wave_sum_dpp(sa_exp2((y0 - b) * c) + sa_exp2((y1 - b) * c));
            const float ht = TWO ? sa_wave_sum_dpp(sa_exp2((y0 - b) * SA_LOG2E) + sa_exp2((y1 - b) * SA_LOG2E)) : st;
            if (lane == 0) { list[0] = mt; list[1] = st; list[2] = ht; }
        }
        if (lane == 0) { list[3] = qr; soft_row = soft; }
    }

    // the student: all tokens, or those that are not in the list
    DisSum d{-INFINITY, 0.0f, 0.0f};
    auto marks = [&](int v) { return (bitmap[v >> 5] >> (v & 31)) & ((1u << VEC) - 1u); };
    auto drop = [&](uint4& r, int q0) {
        const unsigned bits = marks(q0 * VEC);
        if (bits) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if ((bits >> e) & 1u) sa_drop_element<T>(r, e);
        }
    };
    auto power = [](float e) { return HARD == 2 ? e * e : (e * e) * (e * e); };
    // (the logits of two bytes are widened again for every use: kept as they are, they would take twice the registers)
    auto again = [](uint4& r) {
        if constexpr (sizeof(T) == 2 && !KEEP) asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * NT < nq) {
            if (REST && i * NT + tid < nq) drop(raw[i], i * NT + tid);
#pragma unroll
            for (int e = 0; e < VEC; ++e) d.m = fmaxf(d.m, sa_element<T>(raw[i], e));
            again(raw[i]);
        }
    }
    const float own = d.m, bt = dis_base(own);
    float kept[KEEP ? NV * VEC : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * NT < nq) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = sa_element<T>(raw[i], e) - bt, u = sa_exp2(t * c);
                d.s += u;
                if (HARD == 1) d.h += sa_exp2(t * SA_LOG2E);
                if (HARD > 1) d.h += power(u);
                if (KEEP) kept[i * VEC + e] = u;
            }
            again(raw[i]);
        }
    }
    // what the registers do not hold: the next `stash` vectors of a thread stay in LDS, the others are read again
    for (int i = NV; MORE && i * NT < nq; i += 4) {
        uint4 r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = sa_load_vec(xr, ((i + u) * NT + tid) * VEC - lead, V);
        float m = d.m;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (REST && (i + u) * NT + tid < nq) drop(r[u], (i + u) * NT + tid);
            if (i + u - NV < stash) held[(i + u - NV) * NT + tid] = r[u];
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = fmaxf(m, sa_element<T>(r[u], e));
        }
        const float b = dis_base(m), o = d.m - b;
        d.s *= sa_exp2(o * c);
        if (TWO) d.h *= sa_exp2(o * SA_LOG2E);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = sa_element<T>(r[u], e) - b, g = sa_exp2(t * c);
                d.s += g;
                if (HARD == 1) d.h += sa_exp2(t * SA_LOG2E);
                if (HARD > 1) d.h += power(g);
            }
        d.m = m;
    }
    {   // the wave, then the waves in their order
        const float m = sa_wave_max_dpp(d.m), o = d.m - dis_base(m);
        d.s = sa_wave_sum_dpp(d.s * sa_exp2(o * c));
        d.h = TWO ? sa_wave_sum_dpp(d.h * sa_exp2(o * SA_LOG2E)) : d.s;
        d.m = m;
    }
    if (lane == 0) waves[tid >> 6] = d;
    __syncthreads();
    float mr = waves[0].m, sr = 0.0f, hr = 0.0f;
#pragma unroll
    for (int i = 1; i < NW; ++i) mr = fmaxf(mr, waves[i].m);
    const float br = dis_base(mr);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const float o = waves[i].m - br;
        sr += waves[i].s * sa_exp2(o * c);
        if (TWO) hr += waves[i].h * sa_exp2(o * SA_LOG2E);
    }
    if (!TWO) hr = sr;
    // over all tokens, relative to m
    float m = mr, S = sr, H = hr, pr = 1.0f, ph = 1.0f;
    if (REST) {
        m = fmaxf(mr, list[0]);
        const float b = dis_base(m), t = list[0] - b, o = mr - b;
        const float er = sa_exp2(o * c), eh = TWO ? sa_exp2(o * SA_LOG2E) : er;
        S = sr * er + list[1] * sa_exp2(t * c);
        H = TWO ? hr * eh + list[2] * sa_exp2(t * SA_LOG2E) : S;
        pr = sr == 0.0f ? 0.0f : sr * er / S;   // the student's p of the rest, at T and at 1
        ph = hr == 0.0f ? 0.0f : hr * eh / H;
        qr = list[3];
    }
    soft = soft_row != 0;

    if (A.loss_rows && tid < 64) {
        const float lS = logf(S);
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (q[i] != 0.0f) l += q[i] * ((a[i] - am) - lt - ((xv[i] - m) / A.temperature - lS));
        l = sa_wave_sum_dpp(l);
        if (lane == 0) {
            if (REST && qr != 0.0f) l += qr * ((ar - am) - lt - ((mr - m) / A.temperature + logf(sr) - lS));
            float v = soft ? A.alpha * A.temperature * A.temperature * l : 0.0f;
            if (hard) v += (1.0f - A.alpha) * (logf(H) - (xt - m));
            A.loss_rows[row] = f * v;
        }
    }
    if (!dr) return;
    // the gradient: a row-wide formula for the tokens that are not in the list -- relative to THEIR maximum, so that nothing
    // overflows where the list is far above them: p_v = p_rest r_v with r = softmax over the rest --, then the list and the target
    const float cs = soft ? f * A.alpha * A.temperature : 0.0f, ch = hard ? f * (1.0f - A.alpha) : 0.0f;
    const bool live = cs != 0.0f || ch != 0.0f;  // (a row without a list and without a target: zeros, whatever it holds)
    float kr = sr == 0.0f ? 0.0f : cs * (REST ? pr - qr : 1.0f) / sr, kh = hr == 0.0f ? 0.0f : ch * ph / hr;
    if (!TWO) kr += kh;
    if (!live) {
        const float zero[VEC] = {};
        for (int p = tid; p < nq; p += NT) sa_store_vec<T>(dr, p * VEC - lead, V, zero, aligned);
        return;
    }
    auto grad = [&](uint4& r, int q0) {
        float g[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float t = sa_element<T>(r, e) - br, u = sa_exp2(t * c);
            g[e] = kr * u;
            if (HARD == 1) g[e] += kh * sa_exp2(t * SA_LOG2E);
            if (HARD > 1) g[e] += kh * power(u);
        }
        sa_store_vec<T>(dr, q0 * VEC - lead, V, g, aligned);
    };
    // (the kept exponentials are relative to the thread's own maximum; a thread without a finite one kept zeros)
    const float shift = own == -INFINITY ? 0.0f : sa_exp2((bt - br) * c), krt = kr * shift, kht = HARD > 1 ? kh * power(shift) : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int p = i * NT + tid;
        if (p >= nq) continue;
        if constexpr (KEEP) {
            float g[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float u = kept[i * VEC + e];
                g[e] = HARD > 1 ? krt * u + kht * power(u) : krt * u;
            }
            sa_store_vec<T>(dr, p * VEC - lead, V, g, aligned);
        } else {
            grad(raw[i], p);
        }
    }
    for (int i = NV; MORE && i * NT < nq; i += 4) {
        uint4 r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            r[u] = i + u - NV < stash ? held[(i + u - NV) * NT + tid] : sa_load_vec(xr, ((i + u) * NT + tid) * VEC - lead, V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if ((i + u) * NT + tid < nq) grad(r[u], (i + u) * NT + tid);
    }
    __syncthreads();
    if (tid < 64) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (first[i]) {
                const float t = xv[i] - m;
                const float g = cs * (sa_exp2(t * c) / S - qsum[i]) + (hard ? ch * (sa_exp2(t * SA_LOG2E) / H - (id[i] == target ? 1.0f : 0.0f)) : 0.0f);
                dr[id[i]] = sa_narrow<T>(g);
            }
        if (lane == 0 && hard && !((bitmap[(target + lead) >> 5] >> ((target + lead) & 31)) & 1u)) {
            const float t = xt - br;
            const float g = (TWO ? kr * sa_exp2(t * c) + kh * sa_exp2(t * SA_LOG2E) : kr * sa_exp2(t * c)) - ch;
            dr[target] = sa_narrow<T>(g);
        }
    }
}

// *loss = the sum of the rows' losses, in a fixed order and in 64 bits
__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* __restrict__ rows, long n, float* __restrict__ loss) {
    __shared__ double part[16];
    double s = 0.0;
    for (long i = threadIdx.x; i < n; i += 1024) s += (double)rows[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += part[w];
        *loss = (float)s;
    }
}

template <typename T, int NT, int NV, bool MORE, bool REST, int HARD>
bool dis_run(const void* x, void* dx, const SaRows& at, long rows, int V, const DisArgs& A, hipStream_t stream) {
    // rows beyond the registers: as many vectors as 152 KB of LDS hold beside the bitmap
    const size_t bits = (size_t)((V + 2 * SaVec<T>::N + 31) / 32) * 4;
    const int more = (V + 2 * SaVec<T>::N - 2) / SaVec<T>::N - NT * NV;
    int stash = MORE && more > 0 ? (int)((152 * 1024 - bits) / (16 * NT)) : 0;
    if (stash * NT > more) stash = more > 0 ? (more + NT - 1) / NT : 0;
    const size_t smem = bits + (size_t)stash * NT * 16;
    constexpr auto kernel = distill_kernel<T, NT, NV, MORE, REST, HARD>;
    if (smem > 48 * 1024 &&
        hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
        return false;
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(NT), smem, stream, (const T*)x, (T*)dx, at, V, stash, A);
    return true;
}

template <typename T, int NT, int NV, bool MORE, bool REST>
bool dis_hard(const void* x, void* dx, const SaRows& at, long rows, int V, const DisArgs& A, hipStream_t stream) {
    if (A.alpha == 1.0f || !A.targets || A.temperature == 1.0f) return dis_run<T, NT, NV, MORE, REST, 0>(x, dx, at, rows, V, A, stream);
    if (A.temperature == 2.0f) return dis_run<T, NT, NV, MORE, REST, 2>(x, dx, at, rows, V, A, stream);
    if (A.temperature == 4.0f) return dis_run<T, NT, NV, MORE, REST, 4>(x, dx, at, rows, V, A, stream);
    return dis_run<T, NT, NV, MORE, REST, 1>(x, dx, at, rows, V, A, stream);
}

template <typename T, int NT, int NV, bool MORE = false>
bool dis_pick(const void* x, void* dx, const SaRows& at, long rows, int V, const DisArgs& A, hipStream_t stream) {
    return A.rest ? dis_hard<T, NT, NV, MORE, true>(x, dx, at, rows, V, A, stream)
                  : dis_hard<T, NT, NV, MORE, false>(x, dx, at, rows, V, A, stream);
}

// The smallest workgroup whose registers hold a row, 64 exponentials a thread at most: up to 128 registers a thread, so that the
// 512-thread ones run two to a CU and one stores while the other loads (4096 x 32000 bf16: 110 us with 512 threads, 134 with 256,
// 185 with 1024; recomputing the exponentials from 16-bit logits takes a third of the registers and 124 us).  A row beyond that
// keeps what it can in LDS: 1024 threads, 256 KB in registers and 128 KB in LDS (2048 x 131072 f32: 440 us; without LDS 534, two
// smaller workgroups on a CU 580 - 615, all of them bound by what is read twice).  A short row is one wave's, without any exchange
// (16000 x 1000 f32: 31 us against 54 with 256 threads, 8000 x 2000 bf16: 24.5 against 41.6).
struct DisForm { int nt, nv; bool more; };  // threads, vectors a thread holds in registers, rows beyond that
DisForm dis_form(int V, int vec) {
    const int vectors = (V + 2 * vec - 2) / vec;  // of the longest row, with its lead
    if (vectors <= 64 * 2) return {64, 2, false};
    if (vectors <= 64 * 4) return {64, 4, false};
    if (vectors <= 256 * 4) return {256, 4, false};
    if (vectors <= 512 * 32 / vec) return {512, 32 / vec, false};
    if (vectors <= 512 * 64 / vec) return {512, 64 / vec, false};
    return {1024, 64 / vec, vectors > 1024 * 64 / vec};
}
template <typename T>
bool dis_launch(const void* x, void* dx, const SaRows& at, long rows, int V, const DisArgs& A, hipStream_t stream) {
    constexpr int VEC = SaVec<T>::N;
    const DisForm f = dis_form(V, VEC);
    if (f.nt == 64 && f.nv == 2) return dis_pick<T, 64, 2>(x, dx, at, rows, V, A, stream);
    if (f.nt == 64) return dis_pick<T, 64, 4>(x, dx, at, rows, V, A, stream);
    if (f.nt == 256) return dis_pick<T, 256, 4>(x, dx, at, rows, V, A, stream);
    if (f.nt == 512 && f.nv == 32 / VEC) return dis_pick<T, 512, 32 / VEC>(x, dx, at, rows, V, A, stream);
    if (f.nt == 512) return dis_pick<T, 512, 64 / VEC>(x, dx, at, rows, V, A, stream);
    if (!f.more) return dis_pick<T, 1024, 64 / VEC>(x, dx, at, rows, V, A, stream);
    return dis_pick<T, 1024, 64 / VEC, true>(x, dx, at, rows, V, A, stream);
}

}  // namespace

extern "C" ctcStatus_t sa_distill_loss(const void* x, void* dx, long ld_outer, long ld_inner, int n_inner, int dtype, long rows,
                                       int V, const float* values, const long long* ids, const float* rest, int k,
                                       const long long* targets, const float* weights, float temperature, float alpha,
                                       float scale, const float* d_factor, int skip_unit, float* loss_rows, float* loss,
                                       void* stream_) {
    SA_CLEAR_ERR();
    if (rows < 0 || rows > 0x7fffffffL || n_inner < 1 || !sa_rows_ok(dtype, V) || k < 1 || k > SA_TOP_MAX ||
        !sa_temperature_ok(temperature) || !(alpha >= 0.f && alpha <= 1.f) || (rows > 0 && !loss && !dx) ||
        (loss && !loss_rows && rows > 0))
        return CTC_STATUS_INVALID_VALUE;
    if (!sa_threads_ok(rows, dis_form(V, dtype == SA_F32 ? 4 : 8).nt)) return CTC_STATUS_INVALID_VALUE;
    hipStream_t stream = (hipStream_t)stream_;
    if (rows > 0) {
        if (!x || !values || !ids) return CTC_STATUS_INVALID_VALUE;
        const SaRows at{ld_outer, ld_inner, n_inner};
        const DisArgs A{values, ids, rest, k, targets, weights, temperature, alpha, scale, d_factor, loss ? 0 : skip_unit,
                        loss ? loss_rows : nullptr};
        const bool ok = dtype == SA_F32    ? dis_launch<float>(x, dx, at, rows, V, A, stream)
                        : dtype == SA_BF16 ? dis_launch<SaBf16>(x, dx, at, rows, V, A, stream)
                                           : dis_launch<SaF16>(x, dx, at, rows, V, A, stream);
        if (!ok) return CTC_STATUS_EXECUTION_FAILED;
    }
    if (loss) hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, stream, (const float*)loss_rows, rows, loss);
    SA_CHECK_LAUNCH();
    return CTC_STATUS_SUCCESS;
}
