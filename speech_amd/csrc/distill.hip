// distill.hip -- distillation from a teacher's top logits, loss and gradient (sa_distill_loss; the formulas are in
// include/speech_amd.h).
//
// exp2((x - m) log2 e / T) with the maximum subtracted FIRST: the difference of two close numbers is exact, and a row that is masked
// with the type's lowest value stays finite (a fused x c - m c would leave the rounding error of m c, which is huge there).
// The listed tokens and the rest have maxima and sums of their own: p_rest is a sum of its own terms and no difference from 1, and
// it does not vanish when the rest lies far below the list.
#include "rows.h"

namespace {

constexpr int kDisThreads = 256, kDisWaves = kDisThreads / 64;

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

template <typename T>
__global__ __launch_bounds__(kDisThreads) void distill_kernel(const T* __restrict__ x, T* dx, SaRows at, int V, DisArgs A) {
    extern __shared__ unsigned bitmap[];  // V bits: the token is in the list
    __shared__ float scratch[kDisWaves];
    __shared__ int ids[SA_TOP_MAX];
    __shared__ float q[SA_TOP_MAX];
    const long row = blockIdx.x;
    const int tid = threadIdx.x;
    float f = A.scale;
    if (A.factor) {
        if (A.skip_unit && *A.factor == 1.0f) return;
        f *= *A.factor;
    }
    const float w = A.weights ? A.weights[row] : 1.0f;
    const T* xr = x + at.at(row);
    T* dr = dx ? dx + at.at(row) : nullptr;
    if (w == 0.0f) {  // nothing of the row is read: it may hold anything
        if (dr)
            for (int v = tid; v < V; v += kDisThreads) dr[v] = sa_narrow<T>(0.0f);
        if (A.loss_rows && tid == 0) A.loss_rows[row] = 0.0f;
        return;
    }
    f *= w;

    // the teacher: log q and q of the list and of the rest
    for (int i = tid; i < (V + 31) / 32; i += kDisThreads) bitmap[i] = 0;
    __syncthreads();
    int id = -1;
    float a = -INFINITY;
    if (tid < A.k) {
        const long long t = A.ids[row * A.k + tid];
        if (t >= 0 && t < V) {
            id = (int)t;
            a = A.values[row * A.k + tid] / A.temperature;
            atomicOr(&bitmap[id >> 5], 1u << (id & 31));
        }
        ids[tid] = id;
    }
    const bool resting = A.rest != nullptr;
    const float ar = resting ? A.rest[row] : -INFINITY;
    const float am = fmaxf(sa_block_max<kDisWaves>(a, scratch), ar);
    const bool soft = am > -INFINITY && A.alpha > 0.0f;
    const float e = soft ? sa_exp2((a - am) * SA_LOG2E) : 0.0f, er = soft && resting ? sa_exp2((ar - am) * SA_LOG2E) : 0.0f;
    const float total = sa_block_sum<kDisWaves>(e, scratch) + er;
    const float lt = logf(total), qj = soft ? e / total : 0.0f, qr = soft ? er / total : 0.0f;
    if (tid < A.k) q[tid] = qj;
    __syncthreads();

    // the student: maxima and sums over the list (first occurrence of an id) and over the others
    bool first = id >= 0;
    float qsum = 0.0f;  // over the entries of the same id
    if (id >= 0)
        for (int j = 0; j < A.k; ++j)
            if (ids[j] == id) {
                if (j < tid) first = false;
                qsum += q[j];
            }
    const float c = SA_LOG2E / A.temperature;
    const float xv = id >= 0 ? sa_widen(xr[id]) : -INFINITY;
    float mr = -INFINITY;
    for (int v = tid; v < V; v += kDisThreads)
        if (!((bitmap[v >> 5] >> (v & 31)) & 1u)) mr = fmaxf(mr, sa_widen(xr[v]));
    mr = sa_block_max<kDisWaves>(mr, scratch);
    const float mt = sa_block_max<kDisWaves>(first ? xv : -INFINITY, scratch);
    const float m = fmaxf(mr, mt);
    const bool hard_on = A.alpha < 1.0f && A.targets;
    float sr = 0.0f, hr = 0.0f;
    for (int v = tid; v < V; v += kDisThreads)
        if (!((bitmap[v >> 5] >> (v & 31)) & 1u)) {
            const float d = sa_widen(xr[v]) - mr;
            sr += sa_exp2(d * c);
            hr += sa_exp2(d * SA_LOG2E);
        }
    if (mr == -INFINITY) sr = hr = 0.0f;
    sr = sa_block_sum<kDisWaves>(sr, scratch);
    hr = sa_block_sum<kDisWaves>(hr, scratch);
    const float st = sa_block_sum<kDisWaves>(first ? sa_exp2((xv - mt) * c) : 0.0f, scratch);
    const float ht = sa_block_sum<kDisWaves>(first ? sa_exp2((xv - mt) * SA_LOG2E) : 0.0f, scratch);
    // over all tokens, relative to m
    const float S = (mr > -INFINITY ? sr * sa_exp2((mr - m) * c) : 0.0f) + (mt > -INFINITY ? st * sa_exp2((mt - m) * c) : 0.0f);
    const float H = (mr > -INFINITY ? hr * sa_exp2((mr - m) * SA_LOG2E) : 0.0f) +
                    (mt > -INFINITY ? ht * sa_exp2((mt - m) * SA_LOG2E) : 0.0f);
    const float lS = logf(S), lH = logf(H);
    const float logpr = (mr - m) / A.temperature + logf(sr) - lS;

    const long long target = hard_on ? A.targets[row] : -1;
    const bool hard = target >= 0 && target < V;
    if (A.loss_rows) {
        float l = qj > 0.0f ? qj * ((a - am) - lt - ((xv - m) / A.temperature - lS)) : 0.0f;
        l = sa_block_sum<kDisWaves>(l, scratch);
        if (tid == 0) {
            if (qr > 0.0f) l += qr * ((ar - am) - lt - logpr);
            float v = soft ? A.alpha * A.temperature * A.temperature * l : 0.0f;
            if (hard) v += (1.0f - A.alpha) * (lH - (sa_widen(xr[target]) - m));
            A.loss_rows[row] = f * v;
        }
    }
    if (!dr) return;
    // the gradient: a row-wide formula for the tokens that are not in the list -- relative to THEIR maximum, so that nothing
    // overflows where the list is far above them: p_v = p_rest r_v with r = softmax over the rest --, then the list
    const float cs = soft ? f * A.alpha * A.temperature : 0.0f, ch = hard ? f * (1.0f - A.alpha) : 0.0f;
    const float pr = sr == 0.0f ? 0.0f : sr * sa_exp2((mr - m) * c) / S;
    const float kr = sr == 0.0f ? 0.0f : cs * (pr - qr) / sr, kh = hr == 0.0f ? 0.0f : ch * sa_exp2((mr - m) * SA_LOG2E) / H;
    const float base = mr > -INFINITY ? mr : 0.0f;
    for (int v = tid; v < V; v += kDisThreads)
        if (!((bitmap[v >> 5] >> (v & 31)) & 1u)) {
            const float d = sa_widen(xr[v]) - base;
            const float g = kr * sa_exp2(d * c) + kh * sa_exp2(d * SA_LOG2E) - (v == target ? ch : 0.0f);
            dr[v] = sa_narrow<T>(g);
        }
    if (first) {
        const float d = xv - m;
        const float g = cs * (sa_exp2(d * c) / S - qsum) + ch * sa_exp2(d * SA_LOG2E) / H - (id == target ? ch : 0.0f);
        dr[id] = sa_narrow<T>(g);
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

template <typename T>
bool dis_launch(const void* x, void* dx, const SaRows& at, long rows, int V, const DisArgs& A, hipStream_t stream) {
    const size_t smem = (size_t)((V + 31) / 32) * 4;
    if (smem > 48 * 1024 && hipFuncSetAttribute((const void*)distill_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                (int)smem) != hipSuccess)
        return false;
    hipLaunchKernelGGL((distill_kernel<T>), dim3((unsigned)rows), dim3(kDisThreads), smem, stream, (const T*)x, (T*)dx, at, V, A);
    return true;
}

}  // namespace

extern "C" ctcStatus_t sa_distill_loss(const void* x, void* dx, long ld_outer, long ld_inner, int n_inner, int dtype, long rows,
                                       int V, const float* values, const long long* ids, const float* rest, int k,
                                       const long long* targets, const float* weights, float temperature, float alpha,
                                       float scale, const float* d_factor, int skip_unit, float* loss_rows, float* loss,
                                       void* stream_) {
    SA_CLEAR_ERR();
    if (rows < 0 || rows > 0x7fffffffL || n_inner < 1 || !sa_rows_ok(dtype, V) || k < 1 || k > SA_TOP_MAX ||
        !(temperature > 0.f) || !(temperature < INFINITY) || !(alpha >= 0.f && alpha <= 1.f) || (rows > 0 && !loss && !dx) ||
        (loss && !loss_rows && rows > 0))
        return CTC_STATUS_INVALID_VALUE;
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
