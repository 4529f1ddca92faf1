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
// One wave per row. Lane j holds drafted key j's score (its key row read whole, the query's quants from LDS), then lane l
// holds the dims (HD / 64) l .. of O.
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

template <int HD, int FMT> __global__ __launch_bounds__(256) void tree_kernel(const TreeArgs a) {
    constexpr int N = HD / 64, NBLK = HD / 32, BB = FMT == 1 ? 34 : FMT == 2 ? 18 : 64;
    // a wave's query: int8 quants and block scales (quantized K), or fp16 values
    __shared__ __attribute__((aligned(16))) uint32_t qs[4][HD / 2];
    __shared__ float qd[4][NBLK], qsum[4][NBLK];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t r = blockIdx.x * 4 + wave;                        // output row h * rows + i
    if (r >= a.m.nkv * a.m.rows) return;
    const uint32_t h = r / a.m.rows, i = r % a.m.rows, nn = a.n_nodes;
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
                qs[wave][(N * lane + k) / 2] = pa_as_u32(v);
            }
        } else {                                                     // quantize_row_q8_0_ref
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
                ((int8_t *) qs[wave])[N * lane + k] = (int8_t) v;
            }
            #pragma unroll
            for (int off = 1; off < 32 / N; off <<= 1) s += __shfl_xor(s, off);
            if (lane % (32 / N) == 0) { qd[wave][lane / (32 / N)] = (float) (_Float16) d; qsum[wave][lane / (32 / N)] = -8.0f * (float) s; }
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");       // one wave's LDS operations run in order
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
                for (int c = 0; c < 16; c++) {
                    const pa_h2 kv = pa_as_h2(pa_ld<uint32_t>(k + 64 * b + 4 * c)), qv = pa_as_h2(qs[wave][16 * b + c]);
                    t = fmaf((float) kv[0], (float) qv[0], t);
                    t = fmaf((float) kv[1], (float) qv[1], t);
                }
            } else {
                const float d = pa_f16_bits_to_f32(pa_ld<uint16_t>(k + BB * b));
                int dot = 0;
                float off = 0.0f;
                if constexpr (FMT == 1) {
                    #pragma unroll
                    for (int c = 0; c < 8; c++)
                        dot = __builtin_amdgcn_sdot4((int) pa_ld<uint32_t>(k + BB * b + 2 + 4 * c), (int) qs[wave][8 * b + c], dot, false);
                } else {                                             // nibbles as they are: element + 8
                    #pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint32_t w = pa_ld<uint32_t>(k + BB * b + 2 + 4 * c);
                        dot = __builtin_amdgcn_sdot4((int) (w & 0x0f0f0f0fu), (int) qs[wave][8 * b + c], dot, false);
                        dot = __builtin_amdgcn_sdot4((int) ((w >> 4) & 0x0f0f0f0fu), (int) qs[wave][8 * b + 4 + c], dot, false);
                    }
                    off = qsum[wave][b];
                }
                t = fmaf(((float) dot + off) * qd[wave][b], d, t);
            }
        }
        s = t * (a.scale * PA_LOG2E);
    }

    // ---- the slots' statistics, 64 at a time (lane c: slot c), and the common maximum
    const size_t pr = ((size_t) h * a.m.qr + i) * a.m.rst;
    float M = s;
    for (uint32_t c = lane; c < a.m.n_slots; c += 64) M = fmaxf(M, a.m.pml[c * a.m.sst + pr].x);
    M = tr_wavemax(M);
    const float Ms = M == -INFINITY ? 0.0f : M;
    const float p = __builtin_amdgcn_exp2f(s - Ms);
    float L = p, acc[N];
    #pragma unroll
    for (int k = 0; k < N; k++) acc[k] = 0.0f;
    for (uint32_t c0 = 0; c0 < a.m.n_slots; c0 += 64) {
        const float2 ml = c0 + lane < a.m.n_slots ? a.m.pml[(c0 + lane) * a.m.sst + pr] : make_float2(-INFINITY, 0.0f);
        const float w = __builtin_amdgcn_exp2f(ml.x - Ms);           // -inf (an empty or absent slot) -> 0
        L += w * ml.y;
        const uint32_t nc = min(64u, a.m.n_slots - c0);
        for (uint32_t c = 0; c < nc; c++) {
            const float wc = __shfl(w, (int) c);
            const float * o = a.m.po + ((c0 + c) * a.m.sst + pr) * HD + N * lane;
            #pragma unroll
            for (int k = 0; k < N; k++) acc[k] = fmaf(wc, o[k], acc[k]);
        }
    }
    L = tr_wavesum(L);

    // ---- the drafted values: lane l's dims N l .. of each key the row sees
    for (uint64_t left = sees; left; left &= left - 1) {
        const int j = __builtin_ctzll(left);
        const float pj = __shfl(p, j);
        const uint8_t * v = a.v[j] + hoff;
        const int d0 = N * lane, b = d0 / 32, e = d0 % 32;
        float x[N];
        if constexpr (FMT == 0) {
            #pragma unroll
            for (int k = 0; k < N; k++) x[k] = pa_f16_bits_to_f32(pa_ld<uint16_t>(v + 2 * (d0 + k)));
        } else {
            const float d = pa_f16_bits_to_f32(pa_ld<uint16_t>(v + BB * b));
            #pragma unroll
            for (int k = 0; k < N; k++) {
                if constexpr (FMT == 1) x[k] = d * (float) (int8_t) v[BB * b + 2 + e + k];
                else x[k] = d * (float) ((int) ((v[BB * b + 2 + (e & 15) + k] >> (e & 16 ? 4 : 0)) & 15) - 8);
            }
        }
        #pragma unroll
        for (int k = 0; k < N; k++) acc[k] = fmaf(pj, x[k], acc[k]);
    }

    // ---- the reply format
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    #pragma unroll
    for (int k = 0; k < N; k++) a.m.Oh[(size_t) r * HD + N * lane + k] = __builtin_bit_cast(uint16_t, (_Float16) (acc[k] * inv));
    if (lane == 0) a.m.lse[r] = L == 0.0f ? -INFINITY : M * PA_LN2 + logf(L);
}

template <int HD> static hipError_t launch_tree_hd(int fmt, const TreeArgs & a, hipStream_t st) {
    const dim3 grid((a.m.nkv * a.m.rows + 3) / 4);
    if (fmt == 0) hipLaunchKernelGGL((tree_kernel<HD, 0>), grid, dim3(256), 0, st, a);
    else if (fmt == 1) hipLaunchKernelGGL((tree_kernel<HD, 1>), grid, dim3(256), 0, st, a);
    else if (fmt == 2) hipLaunchKernelGGL((tree_kernel<HD, 2>), grid, dim3(256), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_tree(int hd, int fmt, const TreeArgs & a, hipStream_t st) {
    return hd == 128 ? launch_tree_hd<128>(fmt, a, st) : hd == 256 ? launch_tree_hd<256>(fmt, a, st) : hipErrorInvalidValue;
}

}  // namespace pa_hip
