// pa_logprobs.hip - what sampled acceptance and scoring read off the logits (pa_hip_logprobs, gfx950): log-sum-exp, log
// probabilities of given ids, entropy and the best alternatives, one pass over the logits. No counterpart in the reference.
//
// With x a logit and c = scale, a part of a row is (m, S, T) = (max x, sum e^(c (x - m)), sum e^(c (x - m)) (x - m)); two parts
// join as M = max(m1, m2), S = sum f_i S_i, T = sum f_i (T_i + S_i (m_i - M)), f_i = e^(c (m_i - M)). Then
//   lse = c M + ln S,  logp(id) = c (x_id - M) - ln S,  entropy = ln S - c T / S
// (every term of T is <= 0 and of the size of its share, so a row sure of one token loses no digits to a difference). S is NaN
// where a logit is NaN or +inf.
//
// Workgroup (row, w) streams its part of a row through registers, LP_SEG values at a time with the next ones in flight, a
// thread's own maximum as the reference of its sums (no lane waits for another); the workgroups of a row join through memory,
// the last one to finish reading the parts in their order (so the result does not depend on which one it is).
//
// The best n_top: a value is a 64-bit key (order of the value, ~id), so the largest key is the largest value and among equal
// ones the lowest id. A floor under the n_top best is kept: a thread whose maximum is not above it has no candidate, which is
// all that most values cost. Candidates collect in LDS; where they might not fit, 64 groups of four threads take their best keys, and
// the n_top-th largest of these is the new floor: at most n_top groups hold keys at or above it, so what is left always fits.
// A candidate's place is the number of larger ones.
#include "pa_attn.h"
#include "pa_common.h"

namespace pa_hip {

typedef unsigned long long lp_key;

constexpr int LP_TOP = 32, LP_NV = 16, LP_SEG = 256 * LP_NV;
constexpr int LP_CAP = LP_TOP * 4 * LP_NV + LP_TOP;                  // candidates in LDS
static_assert(LP_MAX_PARTS * LP_TOP <= LP_CAP, "the join takes every workgroup's best");

__device__ __forceinline__ uint32_t lp_order(float x) {              // NaN above everything, -0 == +0
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    if (u == 0x80000000u) u = 0u;
    return x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ lp_key lp_make_key(float x, uint32_t idx) { return ((lp_key) lp_order(x) << 32) | (0xffffffffu - idx); }
__device__ __forceinline__ float lp_key_value(lp_key k) {
    const uint32_t u = (uint32_t) (k >> 32);
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);   // (of a NaN's key: a NaN)
}

struct LpPart { float m, s, t; };

__device__ __forceinline__ LpPart lp_join(const LpPart & a, const LpPart & b, float c2) {   // c2 = scale * log2 e
    LpPart r;
    r.m = fmaxf(a.m, b.m);
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
        p = lp_join(p, o, c2);
    }
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = p;
    __syncthreads();
    return lp_join(lp_join(red[0], red[1], c2), lp_join(red[2], red[3], c2), c2);
}

// Loads and conversion of LP_NV values per thread: VEC consecutive ones 256 * VEC apart, as 16-byte buffer loads whose range ends with
// the row's part (any alignment: what lies past the range reads 0 and becomes -inf)
template <typename T> struct LpLoad {
    static constexpr int VEC = 16 / (int) sizeof(T), NL = LP_NV / VEC;
    static __device__ __forceinline__ uint32_t at(int i) { return (uint32_t) ((i / VEC) * 256 * VEC + threadIdx.x * VEC + i % VEC); }
    static __device__ __forceinline__ void load(pa_u4 (&r)[NL], const T * x, uint32_t n) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *) x, (short) 0, (int) (n * sizeof(T)), 0x00020000);
        #pragma unroll
        for (int u = 0; u < NL; u++)
            r[u] = __builtin_bit_cast(pa_u4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (u * 256 + threadIdx.x) * 16, 0, 0));
    }
    static __device__ __forceinline__ float value(T x);
    static __device__ __forceinline__ void convert(const pa_u4 (&r)[NL], const T * x, uint32_t n, float (&v)[LP_NV]) {
        #pragma unroll
        for (int i = 0; i < LP_NV; i++) {
            const uint32_t w = r[i / VEC][sizeof(T) == 4 ? i % VEC : (i % VEC) / 2];
            if constexpr (sizeof(T) == 4) v[i] = __builtin_bit_cast(float, w);
            else v[i] = value(__builtin_bit_cast(T, (uint16_t) (i & 1 ? w >> 16 : w)));
        }
        if (n < (uint32_t) LP_SEG) {
            // (a 16-bit value that ends the range in the middle of a dword is not in reach of its load)
            const float last = sizeof(T) == 2 && (n & 1) ? value(x[n - 1]) : 0.0f;
            #pragma unroll
            for (int i = 0; i < LP_NV; i++) {
                if (sizeof(T) == 2 && (n & 1) && at(i) == n - 1) v[i] = last;
                if (at(i) >= n) v[i] = -INFINITY;
            }
        }
    }
};
template <> __device__ __forceinline__ float LpLoad<float>::value(float x) { return x; }
template <> __device__ __forceinline__ float LpLoad<_Float16>::value(_Float16 x) { return (float) x; }
template <> __device__ __forceinline__ float LpLoad<uint16_t>::value(uint16_t x) { return __builtin_bit_cast(float, (uint32_t) x << 16); }

struct LpShared {
    __attribute__((aligned(16))) lp_key cand[LP_CAP];
    __attribute__((aligned(16))) lp_key wbest[4][64], gbest[4][64];
    lp_key out[LP_TOP];
    LpPart red[4];
    int count;
    bool last;
};

// The n-th largest of the 64 groups' best keys (group l: lane l of each wave; mine: this thread's best, 0 for none), or 0
// where fewer groups have one. Keys are distinct.
__device__ __forceinline__ lp_key lp_floor(int n, lp_key mine, LpShared & sh) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    sh.wbest[wave][lane] = mine;
    __syncthreads();
    lp_key g = 0;
    #pragma unroll
    for (int w = 0; w < 4; w++) g = sh.wbest[w][lane] > g ? sh.wbest[w][lane] : g;
    sh.gbest[wave][lane] = g;                                        // every wave its own copy, read by it alone
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    int above = 0;
    #pragma unroll 16
    for (int i = 0; i < 64; i++) above += sh.gbest[wave][i] > g;
    const unsigned long long who = __ballot(g != 0 && above == n - 1);
    return who ? sh.gbest[wave][__builtin_ctzll(who)] : 0;
}

// The n best of the cur candidates, in order to sh.out (0 where there are fewer)
__device__ __forceinline__ void lp_select(int n, int cur, LpShared & sh) {
    constexpr int R = (LP_CAP + 255) / 256;
    const int t = threadIdx.x;
    if (cur > 128) {                                                 // few enough to be ranked by comparing all of them
        lp_key k[R], mine = 0;
        #pragma unroll
        for (int i = 0; i < R; i++) {
            k[i] = t + 256 * i < cur ? sh.cand[t + 256 * i] : 0;
            mine = k[i] > mine ? k[i] : mine;
        }
        const lp_key fl = lp_floor(n, mine, sh);                     // (its barrier: every candidate is in registers)
        if (t == 0) sh.count = 0;
        __syncthreads();
        if (mine >= fl)
            #pragma unroll
            for (int i = 0; i < R; i++)
                if (k[i] && k[i] >= fl) sh.cand[atomicAdd(&sh.count, 1)] = k[i];
        __syncthreads();
        cur = sh.count;
    }
    if (t < n) sh.out[t] = 0;
    __syncthreads();
    for (int i = t; i < cur; i += 256) {
        const lp_key k = sh.cand[i];
        int place = 0;
        for (int j = 0; j < cur; j++) place += sh.cand[j] > k;
        if (k && place < n) sh.out[place] = k;
    }
    __syncthreads();
}

template <typename T> __global__ __launch_bounds__(256) void logprob_kernel(const LogprobArgs a) {
    using L = LpLoad<T>;
    __shared__ LpShared sh;
    const int row = blockIdx.x / a.parts, w = blockIdx.x % a.parts, t = threadIdx.x;
    const T * x = (const T *) a.logits + (size_t) row * (size_t) a.stride;
    const uint32_t j0 = (uint32_t) w * a.span, j1 = (uint32_t) min((int64_t) a.vocab, (int64_t) j0 + a.span);
    const float c2 = a.scale * PA_LOG2E;
    LpPart p = {-INFINITY, 0.0f, 0.0f};
    lp_key floor = 0;
    float fval = 0.0f;
    int cur = 0;                                                     // candidates in LDS
    pa_u4 r[L::NL];
    L::load(r, x + j0, min(j1 - j0, (uint32_t) LP_SEG));
    if (t == 0) sh.count = 0;
    for (uint32_t j = j0; j < j1; j += LP_SEG) {
        const uint32_t n = min(j1 - j, (uint32_t) LP_SEG);
        float v[LP_NV];
        L::convert(r, x + j, n, v);
        if (j + LP_SEG < j1) L::load(r, x + j + LP_SEG, min(j1 - j - LP_SEG, (uint32_t) LP_SEG));
        float mt = v[0];
        #pragma unroll
        for (int i = 1; i < LP_NV; i++) mt = fmaxf(mt, v[i]);
        const float m = fmaxf(p.m, mt), ms = m == -INFINITY ? 0.0f : m;
        const float d0 = p.m == -INFINITY ? 0.0f : p.m - m, f = __builtin_amdgcn_exp2f(d0 * c2);
        p.t = f > 0.0f ? (p.t + p.s * d0) * f : 0.0f;
        p.s *= f;
        p.m = m;
        #pragma unroll
        for (int i = 0; i < LP_NV; i++) {
            const float d = v[i] - ms, e = __builtin_amdgcn_exp2f(d * c2);
            p.s += e;
            p.t = fmaf(e, fmaxf(d, -3e38f), p.t);                    // -inf: e = 0, and 0 * (a number) = 0
        }
        if (a.n_top == 0) continue;
        const bool any = L::at(0) < n, nan = p.s != p.s;             // (at(0): this thread's first value)
        auto hits = [&] { return any && (floor == 0 || nan || mt > fval); };
        int h = __syncthreads_count(hits());
        if (h == 0) continue;
        auto each = [&](auto f) {
            #pragma unroll
            for (int i = 0; i < LP_NV; i++)
                if (L::at(i) < n) f(lp_make_key(v[i], j + L::at(i)));
        };
        if (cur + h * LP_NV > LP_CAP) {
            if (cur > 0) {                                           // the n_top best so far, and their last one as the floor
                lp_select(a.n_top, cur, sh);
                if (t < a.n_top) sh.cand[t] = sh.out[t];
                cur = a.n_top;
                const lp_key k = sh.out[a.n_top - 1];
                if (k > floor) { floor = k; fval = lp_key_value(k); }
                if (t == 0) sh.count = cur;
                h = __syncthreads_count(hits());
            }
            if (cur + h * LP_NV > LP_CAP) {
                lp_key mine = 0;
                if (hits()) each([&](lp_key k) { mine = k > mine ? k : mine; });
                const lp_key k = lp_floor(a.n_top, mine, sh);
                if (k > floor) { floor = k; fval = lp_key_value(k); }
            }
        }
        if (any && (floor == 0 || nan || mt >= fval))
            each([&](lp_key k) { if (k >= floor) sh.cand[atomicAdd(&sh.count, 1)] = k; });
        __syncthreads();
        cur = sh.count;
    }
    if (a.n_top > 0) lp_select(a.n_top, cur, sh);
    p = lp_join_all(p, c2, sh.red);

    if (a.parts > 1) {
        // this workgroup's part and best keys, written through and complete before it counts itself done
        float2 * part = (float2 *) a.part + 2 * ((size_t) row * a.parts + w);
        lp_key * keys = a.keys + ((size_t) row * a.parts + w) * a.n_top;
        if (t < a.n_top) __hip_atomic_store(&keys[t], sh.out[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (t < 2)
            __hip_atomic_store((lp_key *) &part[t], __builtin_bit_cast(lp_key, t ? make_float2(p.t, 0.0f) : make_float2(p.m, p.s)),
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t == 0) {
            const unsigned int done = __hip_atomic_fetch_add(&a.counter[row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sh.last = done == (unsigned int) a.parts - 1;
            if (sh.last) __hip_atomic_store(&a.counter[row], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!sh.last) return;
        part = (float2 *) a.part + 2 * (size_t) row * a.parts;
        keys = a.keys + (size_t) row * a.parts * a.n_top;
        p = LpPart{-INFINITY, 0.0f, 0.0f};
        if (t < a.parts) {
            const float2 ms = __builtin_bit_cast(float2, __hip_atomic_load((lp_key *) &part[2 * t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            const float2 tt = __builtin_bit_cast(float2, __hip_atomic_load((lp_key *) &part[2 * t + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            p = LpPart{ms.x, ms.y, tt.x};
        }
        const int nk = a.parts * a.n_top;
        for (int i = t; i < nk; i += 256) sh.cand[i] = __hip_atomic_load(&keys[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        p = lp_join_all(p, c2, sh.red);
        if (a.n_top > 0) lp_select(a.n_top, nk, sh);
    }

    const bool bad = p.s != p.s || p.m == INFINITY, none = p.m == -INFINITY;
    const float ls = logf(p.s);                                      // S >= 1 unless no value is above -inf
    auto logp_of = [&](float v) { return bad ? NAN : none || v == -INFINITY ? -INFINITY : fmaf(v - p.m, a.scale, -ls); };
    if (t == 0) {
        if (a.lse) a.lse[row] = bad ? NAN : none ? -INFINITY : fmaf(p.m, a.scale, ls);
        if (a.entropy) a.entropy[row] = bad ? NAN : none ? 0.0f : ls - a.scale * p.t / p.s;
    }
    for (int i = t; i < a.n_given; i += 256) {
        const int32_t id = a.given[(size_t) row * a.n_given + i];
        a.logp[(size_t) row * a.n_given + i] = id >= 0 && id < a.vocab ? logp_of(L::value(x[id])) : NAN;
    }
    if (t < a.n_top) {
        const lp_key k = sh.out[t];
        a.top_id[(size_t) row * a.n_top + t] = k ? (int32_t) (0xffffffffu - (uint32_t) k) : -1;
        a.top_logp[(size_t) row * a.n_top + t] = k ? logp_of(lp_key_value(k)) : -INFINITY;
    }
}

hipError_t launch_logprobs(const LogprobArgs & a, hipStream_t st) {
    const dim3 grid((uint32_t) a.n_rows * a.parts);
    if (a.n_rows == 0) return hipSuccess;
    if (a.parts > LP_MAX_PARTS || (int64_t) a.parts * a.span < a.vocab || (int64_t) (a.parts - 1) * a.span >= a.vocab) return hipErrorInvalidValue;
    if (a.type == PA_TYPE_F32) hipLaunchKernelGGL(logprob_kernel<float>, grid, dim3(256), 0, st, a);
    else if (a.type == PA_TYPE_F16) hipLaunchKernelGGL(logprob_kernel<_Float16>, grid, dim3(256), 0, st, a);
    else if (a.type == PA_TYPE_BF16) hipLaunchKernelGGL(logprob_kernel<uint16_t>, grid, dim3(256), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace pa_hip
