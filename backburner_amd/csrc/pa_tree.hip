// pa_tree.hip - the last step of a tree attention call (pa_hip_attn_tree, gfx950): the split-K slots of the context before the
// tree joined with the tree's own keys, in the reply format. No counterpart in the reference.
//
// The attention kernels take the context, which every row sees, and leave slots (O unnormalised against the slot's base-2 max,
// max, sum). Here each row adds its softmax over the drafted keys its mask leaves: s_j = scale * q . k_j (ggml's block dots over
// quantized K, fp32 products over f16 K), M = max(slots' max, max_j s_j), then
//   O = sum_c 2^(m_c - M) O_c + sum_j 2^(s_j - M) v_j,  L = sum_c 2^(m_c - M) L_c + sum_j 2^(s_j - M),  Oh = f16(O / L).
// A mask inside the attention kernels would have cost their tile loops a test per tile and a register pair per row, and a
// matrix instruction multiplies a masked key's probability, zero, with whatever its value row holds, where infinities and NaN
// become NaN. Here a value row that a row does not see is never read. At most 64 keys a row: vector work of a few instructions.
//
// W waves per row (1, 4 or 16 by the number of slots), each with every W-th slot and all of its loads issued at once, against its own
// maximum; they meet once, through LDS. Lane l holds the dims (HD / 64) l .. of O. The first wave also takes the drafted keys, lane j
// the score of key j (its key row read whole, the query's quants from LDS); only the ones that the row sees are touched, in a tree
// the few on its path.
//
#include "pa_attn.h"
#include "pa_common.h"

namespace pa_hip {

template <int CTRL> __device__ __forceinline__ float tr_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// max over the 8 or 16 lanes of a quant block (N lanes from a multiple of N on)
template <int N> __device__ __forceinline__ float tr_blockmax(float v) {
    v = fmaxf(v, tr_dpp<0xb1>(v));
    v = fmaxf(v, tr_dpp<0x4e>(v));
    v = fmaxf(v, tr_dpp<0x141>(v));                                  // row_half_mirror: lane ^ 7
    if constexpr (N == 16) v = fmaxf(v, tr_dpp<0x140>(v));           // row_mirror: lane ^ 15
    return v;
}
__device__ __forceinline__ float tr_wavemax(float v) {
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}
__device__ __forceinline__ float tr_wavesum(float v) {
    #pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

template <int HD, int FMT, int W> __global__ __launch_bounds__(W == 16 ? 1024 : 256) void tree_kernel(const TreeArgs a) {
    constexpr int N = HD / 64, NBLK = HD / 32, BB = FMT == 1 ? 34 : FMT == 2 ? 18 : 64, NW = W == 16 ? 16 : 4, RPB = NW / W, S = 16;
    // a row's query: int8 quants and block scales (quantized K), or fp16 values
    __shared__ __attribute__((aligned(16))) uint32_t qs[RPB][HD / 2];
    __shared__ float qd[RPB][NBLK], qsum[RPB][NBLK];
    __shared__ float sm[W > 1 ? W : 1], sl[W > 1 ? W : 1];
    __shared__ __attribute__((aligned(16))) float so[W > 1 ? W : 1][W > 1 ? HD : 1];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wr = wave % W, rb = wave / W;
    const uint32_t r = blockIdx.x * RPB + rb;                        // output row h * rows + i
    if (r >= a.m.nkv * a.m.rows) return;                             // (W > 1: one row per workgroup, so none)
    const uint32_t h = r / a.m.rows, i = r % a.m.rows, nn = a.n_nodes, ns = a.m.n_slots;
    const size_t pr = ((size_t) h * a.m.qr + i) * a.m.rst;

    // ---- a batch of slots: lane u's (max, sum) of slot c0 + W u, and every lane's dims of all of them
    float2 ml;
    float o[S][N];
    auto load_slots = [&](uint32_t c0) {
        const uint32_t c = c0 + W * lane;
        ml = lane < S && c < ns ? a.m.pml[c * a.m.sst + pr] : make_float2(-INFINITY, 0.0f);
        #pragma unroll
        for (int u = 0; u < S; u++) {
            const uint32_t cu = c0 + W * u;
            const float * p = a.m.po + (cu * a.m.sst + pr) * HD + N * lane;
            #pragma unroll
            for (int k = 0; k < N; k++) o[u][k] = 0.0f;
            if (cu < ns) {                                           // uniform
                if constexpr (N == 2) { const float2 x = *(const float2 *) p; o[u][0] = x.x; o[u][1] = x.y; }
                else { const pa_f4 x = *(const pa_f4 *) p; o[u][0] = x[0]; o[u][1] = x[1]; o[u][2] = x[2]; o[u][3] = x[3]; }
            }
        }
    };
    load_slots(wr);

    float m = -INFINITY, L = 0.0f, acc[N];                           // this wave's share, against its own maximum m; L per lane
    #pragma unroll
    for (int k = 0; k < N; k++) acc[k] = 0.0f;
    if (wr == 0) {
        const uint64_t sees = a.mask[i % nn] & (nn < 64 ? (1ull << nn) - 1 : ~0ull);
        const size_t hoff = (size_t) h * a.hb;
        // ---- the query, rounded as the attention kernels round it
        {
            #pragma clang fp contract(off)
            const float * q = a.q + (size_t) r * HD + N * lane;
            float x[N];
            #pragma unroll
            for (int k = 0; k < N; k++) x[k] = q[k];
            if constexpr (FMT == 0) {
                #pragma unroll
                for (int k = 0; k < N; k += 2) {
                    const pa_h2 v = {(_Float16) x[k], (_Float16) x[k + 1]};
                    qs[rb][(N * lane + k) / 2] = pa_as_u32(v);
                }
            } else {                                                 // quantize_row_q8_0_ref
                float am = 0.0f;
                #pragma unroll
                for (int k = 0; k < N; k++) am = fmaxf(am, fabsf(x[k]));
                am = tr_blockmax<32 / N>(am);
                const float d = am / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
                int s = 0;
                #pragma unroll
                for (int k = 0; k < N; k++) {
                    const int v = (int) roundf(x[k] * id);
                    s += v;
                    ((int8_t *) qs[rb])[N * lane + k] = (int8_t) v;
                }
                #pragma unroll
                for (int off = 1; off < 32 / N; off <<= 1) s += __shfl_xor(s, off);
                if (lane % (32 / N) == 0) { qd[rb][lane / (32 / N)] = (float) (_Float16) d; qsum[rb][lane / (32 / N)] = -8.0f * (float) s; }
            }
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");   // one wave's LDS operations run in order
        }
        // ---- lane j: the base-2 score of drafted key j
        float s = -INFINITY;
        if ((sees >> lane) & 1) {
            const uint8_t * k = a.k[lane] + hoff;
            float t = 0.0f;
            #pragma unroll
            for (int b = 0; b < NBLK; b++) {
                if constexpr (FMT == 0) {
                    #pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const pa_u4 kw = pa_ld<pa_u4>(k + 64 * b + 16 * c), qw = *(const pa_u4 *) &qs[rb][16 * b + 4 * c];
                        #pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const pa_h2 kv = pa_as_h2(kw[e]), qv = pa_as_h2(qw[e]);
                            t = fmaf((float) kv[0], (float) qv[0], t);
                            t = fmaf((float) kv[1], (float) qv[1], t);
                        }
                    }
                } else {
                    const float d = pa_f16_bits_to_f32(pa_ld<uint16_t>(k + BB * b));
                    const pa_u4 q0 = *(const pa_u4 *) &qs[rb][8 * b], q1 = *(const pa_u4 *) &qs[rb][8 * b + 4];
                    const pa_u4 k0 = pa_ld<pa_u4>(k + BB * b + 2);
                    pa_u4 w0 = k0, w1;
                    if constexpr (FMT == 1) w1 = pa_ld<pa_u4>(k + BB * b + 18);
                    else { w0 = k0 & 0x0f0f0f0fu; w1 = (k0 >> 4) & 0x0f0f0f0fu; }   // nibbles as they are: element + 8
                    int dot = 0;
                    #pragma unroll
                    for (int c = 0; c < 4; c++) {
                        dot = __builtin_amdgcn_sdot4((int) w0[c], (int) q0[c], dot, false);
                        dot = __builtin_amdgcn_sdot4((int) w1[c], (int) q1[c], dot, false);
                    }
                    t = fmaf(((float) dot + (FMT == 2 ? qsum[rb][b] : 0.0f)) * qd[rb][b], d, t);
                }
            }
            s = t * (a.scale * PA_LOG2E);
        }
        m = tr_wavemax(s);
        const float p = __builtin_amdgcn_exp2f(s - (m == -INFINITY ? 0.0f : m));
        L = p;
        // ---- the drafted values, four at a time: lane l's dims N l .. of each key the row sees
        const int d0 = N * lane, b = d0 / 32, e = d0 % 32;
        for (uint64_t left = sees; left;) {
            float x[4][N], pj[4];
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                const bool is = left != 0;                           // uniform
                const int j = is ? __builtin_ctzll(left) : 0;
                left &= left - 1;
                pj[u] = is ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j)) : 0.0f;
                #pragma unroll
                for (int k = 0; k < N; k++) x[u][k] = 0.0f;
                if (!is) continue;
                const uint8_t * v = a.v[j] + hoff;
                if constexpr (FMT == 0) {
                    #pragma unroll
                    for (int k = 0; k < N; k++) x[u][k] = pa_f16_bits_to_f32(pa_ld<uint16_t>(v + 2 * (d0 + k)));
                } else {
                    const float d = pa_f16_bits_to_f32(pa_ld<uint16_t>(v + BB * b));
                    #pragma unroll
                    for (int k = 0; k < N; k++) {
                        if constexpr (FMT == 1) x[u][k] = d * (float) (int8_t) v[BB * b + 2 + e + k];
                        else x[u][k] = d * (float) ((int) ((v[BB * b + 2 + (e & 15) + k] >> (e & 16 ? 4 : 0)) & 15) - 8);
                    }
                }
            }
            #pragma unroll
            for (int u = 0; u < 4; u++)
                #pragma unroll
                for (int k = 0; k < N; k++) acc[k] = fmaf(pj[u], x[u][k], acc[k]);
        }
    }

    // ---- the slots
    for (uint32_t c0 = wr; c0 < ns;) {
        float mb = ml.x;                                             // lanes 0 .. S - 1
        #pragma unroll
        for (int off = S / 2; off > 0; off >>= 1) mb = fmaxf(mb, __shfl_xor(mb, off));
        mb = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mb)));
        const float mn = fmaxf(m, mb), ms = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f((m == -INFINITY ? ms : m) - ms);   // (nothing yet: acc and L are 0)
        const float w = __builtin_amdgcn_exp2f(ml.x - ms);           // -inf (an empty or absent slot) -> 0
        L = L * f + w * ml.y;
        #pragma unroll
        for (int k = 0; k < N; k++) acc[k] *= f;
        #pragma unroll
        for (int u = 0; u < S; u++) {
            const float wu = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), u));
            #pragma unroll
            for (int k = 0; k < N; k++) acc[k] = fmaf(wu, o[u][k], acc[k]);
        }
        m = mn;
        c0 += W * S;
        if (c0 < ns) load_slots(c0);
    }
    L = tr_wavesum(L);

    // ---- the row's waves
    if constexpr (W > 1) {
        if (lane == 0) { sm[wr] = m; sl[wr] = L; }
        #pragma unroll
        for (int k = 0; k < N; k++) so[wr][N * lane + k] = acc[k];
        __syncthreads();
        if (wr != 0) return;
        float M = sm[0];
        #pragma unroll
        for (int u = 1; u < W; u++) M = fmaxf(M, sm[u]);
        const float Ms = M == -INFINITY ? 0.0f : M;
        float f = __builtin_amdgcn_exp2f((m == -INFINITY ? Ms : m) - Ms);   // (a NaN of the drafted keys stays in acc and L)
        L *= f;
        #pragma unroll
        for (int k = 0; k < N; k++) acc[k] *= f;
        #pragma unroll
        for (int u = 1; u < W; u++) {
            f = __builtin_amdgcn_exp2f(sm[u] - Ms);
            L = fmaf(f, sl[u], L);
            #pragma unroll
            for (int k = 0; k < N; k++) acc[k] = fmaf(f, so[u][N * lane + k], acc[k]);
        }
        m = M;
    }

    // ---- the reply format
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t * out = a.m.Oh + (size_t) r * HD + N * lane;
    if constexpr (N == 2) *(pa_h2 *) out = (pa_h2){(_Float16) (acc[0] * inv), (_Float16) (acc[1] * inv)};
    else *(pa_h4 *) out = (pa_h4){(_Float16) (acc[0] * inv), (_Float16) (acc[1] * inv), (_Float16) (acc[2] * inv), (_Float16) (acc[3] * inv)};
    if (lane == 0) a.m.lse[r] = L == 0.0f ? -INFINITY : m * PA_LN2 + logf(L);
}

template <int HD, int FMT> static void launch_tree_w(const TreeArgs & a, hipStream_t st) {
    const uint32_t rows = a.m.nkv * a.m.rows;
    if (a.m.n_slots <= 16) hipLaunchKernelGGL((tree_kernel<HD, FMT, 1>), dim3((rows + 3) / 4), dim3(256), 0, st, a);
    else if (a.m.n_slots <= 64) hipLaunchKernelGGL((tree_kernel<HD, FMT, 4>), dim3(rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((tree_kernel<HD, FMT, 16>), dim3(rows), dim3(1024), 0, st, a);
}

template <int HD> static hipError_t launch_tree_hd(int fmt, const TreeArgs & a, hipStream_t st) {
    if (fmt == 0) launch_tree_w<HD, 0>(a, st);
    else if (fmt == 1) launch_tree_w<HD, 1>(a, st);
    else if (fmt == 2) launch_tree_w<HD, 2>(a, st);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_tree(int hd, int fmt, const TreeArgs & a, hipStream_t st) {
    return hd == 128 ? launch_tree_hd<128>(fmt, a, st) : hd == 256 ? launch_tree_hd<256>(fmt, a, st) : hipErrorInvalidValue;
}

}  // namespace pa_hip
