// pa_logprobs.hip - what sampled acceptance and scoring read off the logits (pa_hip_logprobs, gfx950): log-sum-exp, log
// probabilities of given ids, entropy and the best alternatives, one pass over the logits. No counterpart in the reference.
//
// With x a logit and c = scale, a part of a row is (m, S, T) = (max x, sum e^(c (x - m)), sum e^(c (x - m)) (x - m)); two parts
// join as M = max(m1, m2), S = sum f_i S_i, T = sum f_i (T_i + S_i (m_i - M)), f_i = e^(c (m_i - M)). Then
//   lse = c M + ln S,  logp(id) = c (x_id - M) - ln S,  entropy = ln S - c T / S
// (every term of T is <= 0 and of the size of its share, so a row sure of one token loses no digits to a difference).
//
// logprob_part_kernel: workgroup (row, split) takes its values into registers, a thread's own maximum as the reference of its sums
// (no lane waits for another), then joins the threads' parts. The best n_top: a value is a 64-bit key (order of the value, ~id),
// so the largest key is the largest value and among equal ones the lowest id. The n_top-th largest of the threads' best keys
// is a floor under the workgroup's n_top best, and at most n_top threads hold keys at or above it, so at most n_top * NV
// candidates are left, typically little more than n_top; each one's place is the number of larger ones.
// logprob_join_kernel: one workgroup per row joins the parts and the keys the same way and reads the given ids' logits.
#include "pa_attn.h"
#include "pa_common.h"

namespace pa_hip {

typedef unsigned long long lp_key;

__device__ __forceinline__ lp_key lp_make_key(float x, uint32_t idx) {   // NaN above everything, -0 == +0, lower ids first
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    if (u == 0x80000000u) u = 0u;
    const uint32_t k = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((lp_key) k << 32) | (0xffffffffu - idx);
}

struct LpPart { float m, s, t; bool nan; };

__device__ __forceinline__ LpPart lp_join(const LpPart & a, const LpPart & b, float c2) {   // c2 = scale * log2 e
    LpPart r;
    r.m = fmaxf(a.m, b.m);
    r.nan = a.nan || b.nan;
    const float da = a.m == -INFINITY ? 0.0f : a.m - r.m, db = b.m == -INFINITY ? 0.0f : b.m - r.m;   // (-inf: s = t = 0)
    const float fa = __builtin_amdgcn_exp2f(da * c2), fb = __builtin_amdgcn_exp2f(db * c2);
    r.s = a.s * fa + b.s * fb;
    // (a part of no weight adds nothing, however far its maximum lies: s * d may overflow there)
    r.t = (fa > 0.0f ? (a.t + a.s * da) * fa : 0.0f) + (fb > 0.0f ? (b.t + b.s * db) * fb : 0.0f);
    return r;
}

// the parts of a workgroup's 256 threads joined; every thread gets the result
__device__ __forceinline__ LpPart lp_join_all(LpPart p, float c2, LpPart (&red)[4]) {
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        LpPart o;
        o.m = __shfl_xor(p.m, off); o.s = __shfl_xor(p.s, off); o.t = __shfl_xor(p.t, off);
        o.nan = __shfl_xor((int) p.nan, off) != 0;
        p = lp_join(p, o, c2);
    }
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = p;
    __syncthreads();
    return lp_join(lp_join(red[0], red[1], c2), lp_join(red[2], red[3], c2), c2);
}

template <typename T> __device__ __forceinline__ float lp_value(const T * x, int64_t i);
template <> __device__ __forceinline__ float lp_value(const float * x, int64_t i) { return x[i]; }
template <> __device__ __forceinline__ float lp_value(const _Float16 * x, int64_t i) { return (float) x[i]; }
template <> __device__ __forceinline__ float lp_value(const uint16_t * x, int64_t i) { return __builtin_bit_cast(float, (uint32_t) x[i] << 16); }

constexpr int LP_TOP = 32;

// The n best of the workgroup's keys (mine: this thread's best; each(f): f(key) for all of this thread's keys at least `floor`),
// in order to out[0 .. n-1] (0 where there are fewer). cand: room for LP_TOP * (keys per thread).
template <class F> __device__ __forceinline__ void lp_select(int n, lp_key mine, F each, lp_key (&best)[256], lp_key * cand, int & count,
                                                             lp_key * out) {
    const int t = threadIdx.x;
    __shared__ lp_key floor_key;
    best[t] = mine;
    if (t == 0) { count = 0; floor_key = 0; }
    if (t < n) out[t] = 0;
    __syncthreads();
    int above = 0;
    for (int i = 0; i < 256; i++) above += best[i] > mine;
    if (above == n - 1 && mine) floor_key = mine;                    // keys are distinct (absent ones are 0)
    __syncthreads();
    const lp_key fl = floor_key;
    if (mine && mine >= fl)
        each([&](lp_key k) { if (k >= fl) cand[atomicAdd(&count, 1)] = k; });
    __syncthreads();
    const int m = count;
    for (int i = t; i < m; i += 256) {
        const lp_key k = cand[i];
        int place = 0;
        for (int j = 0; j < m; j++) place += cand[j] > k;
        if (place < n) out[place] = k;
    }
    __syncthreads();
}

template <typename T, int NV> __global__ __launch_bounds__(256) void logprob_part_kernel(const LogprobArgs a) {
    __shared__ LpPart red[4];
    __shared__ lp_key best[256], cand[LP_TOP * NV], out[LP_TOP];
    __shared__ int count;
    const int row = blockIdx.x / a.splits, sp = blockIdx.x % a.splits, t = threadIdx.x;
    const T * x = (const T *) a.logits + (size_t) row * (size_t) a.stride;
    const int64_t j0 = (int64_t) sp * a.seg;
    const uint32_t n = (uint32_t) min((int64_t) a.seg, a.vocab - j0);
    float v[NV];
    #pragma unroll
    for (int u = 0; u < NV; u++) v[u] = (uint32_t) (t + 256 * u) < n ? lp_value<T>(x, j0 + t + 256 * u) : -INFINITY;
    LpPart p = {-INFINITY, 0.0f, 0.0f, false};
    lp_key mine = 0;
    #pragma unroll
    for (int u = 0; u < NV; u++) {
        p.m = fmaxf(p.m, v[u]);
        p.nan |= v[u] != v[u];
    }
    const float c2 = a.scale * PA_LOG2E;
    if (p.m > -INFINITY) {
        #pragma unroll
        for (int u = 0; u < NV; u++) {
            const float d = fmaxf(v[u] - p.m, -3e38f), e = __builtin_amdgcn_exp2f(d * c2);   // -inf: e = 0, e * d = 0
            p.s += e;
            p.t = fmaf(e, d, p.t);
        }
    }
    p = lp_join_all(p, c2, red);
    if (t == 0) a.part[(size_t) row * a.splits + sp] = make_float4(p.m, p.s, p.t, p.nan ? 1.0f : 0.0f);
    if (a.n_top == 0) return;
    auto each = [&](auto f) {
        #pragma unroll
        for (int u = 0; u < NV; u++)
            if ((uint32_t) (t + 256 * u) < n) f(lp_make_key(v[u], (uint32_t) j0 + t + 256 * u));
    };
    each([&](lp_key k) { mine = k > mine ? k : mine; });
    lp_select(a.n_top, mine, each, best, cand, count, out);
    if (t < a.n_top) a.keys[((size_t) row * a.splits + sp) * a.n_top + t] = out[t];
}

template <typename T> __global__ __launch_bounds__(256) void logprob_join_kernel(const LogprobArgs a) {
    __shared__ LpPart red[4];
    __shared__ lp_key best[256], out[LP_TOP];
    extern __shared__ lp_key cand[];
    __shared__ int count;
    const int row = blockIdx.x, t = threadIdx.x;
    const T * x = (const T *) a.logits + (size_t) row * (size_t) a.stride;
    const float c2 = a.scale * PA_LOG2E;
    LpPart p = {-INFINITY, 0.0f, 0.0f, false};
    for (int i = t; i < a.splits; i += 256) {
        const float4 q = a.part[(size_t) row * a.splits + i];
        p = lp_join(p, LpPart{q.x, q.y, q.z, q.w != 0.0f}, c2);
    }
    p = lp_join_all(p, c2, red);
    const bool bad = p.nan || p.m == INFINITY, none = p.m == -INFINITY;
    const float ls = logf(p.s);                                      // S >= 1 unless no value is above -inf
    auto logp_of = [&](float v) { return bad ? NAN : none || v == -INFINITY ? -INFINITY : fmaf(v - p.m, a.scale, -ls); };
    if (t == 0) {
        if (a.lse) a.lse[row] = bad ? NAN : none ? -INFINITY : fmaf(p.m, a.scale, ls);
        if (a.entropy) a.entropy[row] = bad ? NAN : none ? 0.0f : ls - a.scale * p.t / p.s;
    }
    for (int i = t; i < a.n_given; i += 256) {
        const int32_t id = a.given[(size_t) row * a.n_given + i];
        a.logp[(size_t) row * a.n_given + i] = id >= 0 && id < a.vocab ? logp_of(lp_value<T>(x, id)) : NAN;
    }
    if (a.n_top == 0) return;
    const lp_key * keys = a.keys + (size_t) row * a.splits * a.n_top;
    const int nk = a.splits * a.n_top;
    lp_key mine = 0;
    auto each = [&](auto f) {
        for (int i = t; i < nk; i += 256)
            if (keys[i]) f(keys[i]);
    };
    each([&](lp_key k) { mine = k > mine ? k : mine; });
    lp_select(a.n_top, mine, each, best, cand, count, out);
    if (t < a.n_top) {
        const lp_key k = out[t];
        const int32_t id = k ? (int32_t) (0xffffffffu - (uint32_t) k) : -1;
        a.top_id[(size_t) row * a.n_top + t] = id;
        a.top_logp[(size_t) row * a.n_top + t] = k ? logp_of(lp_value<T>(x, id)) : -INFINITY;
    }
}

template <typename T> static hipError_t launch_logprobs_t(const LogprobArgs & a, hipStream_t st) {
    const dim3 grid((uint32_t) a.n_rows * a.splits);
    if (a.seg == 4096) hipLaunchKernelGGL((logprob_part_kernel<T, 16>), grid, dim3(256), 0, st, a);
    else if (a.seg == 16384) hipLaunchKernelGGL((logprob_part_kernel<T, 64>), grid, dim3(256), 0, st, a);
    else return hipErrorInvalidValue;
    // a thread of the join holds at most ceil(keys / 256) keys, n_top threads of them candidates
    const size_t cand = (size_t) a.n_top * ((a.splits * a.n_top + 255) / 256);
    hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((uint32_t) a.n_rows), dim3(256), cand * sizeof(lp_key), st, a);
    return hipGetLastError();
}

hipError_t launch_logprobs(const LogprobArgs & a, hipStream_t st) {
    if (a.n_rows == 0) return hipSuccess;
    if (a.type == PA_TYPE_F32) return launch_logprobs_t<float>(a, st);
    if (a.type == PA_TYPE_F16) return launch_logprobs_t<_Float16>(a, st);
    if (a.type == PA_TYPE_BF16) return launch_logprobs_t<uint16_t>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace pa_hip
