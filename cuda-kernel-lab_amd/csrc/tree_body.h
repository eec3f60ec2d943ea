// tree_body.h -- attention of drafted tokens over the paged cache (pdattn_tree_attention): several query
// tokens per sequence, seeing the cached keys before them and, of each other, an ancestor mask's or a
// chain's, with scores that may be capped, biased by distance and windowed. Compiled with cascade.hip.
//
//   x = sm_scale q.k;  x = cap tanh(x / cap);  x += slope_h (pos_k - pos_q);  unseen: -inf
//   out = sum_k softmax(x)_k v_k,  lse = ln sum_k exp(x_k)
//
// One wave per (token, query head): 64 keys at a time, a key per lane for the scores, two dims per lane
// for the output.
#pragma once

#include <math.h>

#include "pdattn_internal.h"

namespace pdattn {
namespace {

constexpr float kTreeLn2 = 0.69314718055994531f;
constexpr int kTreeMaxTokens = PDATTN_TREE_MAX_TOKENS;

// tanh(x) in 32 bits. |x| <= 1: the fifth convergent of x / (1 + x^2 / (3 + x^2 / (5 + ...))) (Lambert), of
// which 32 bits show no error; else 1 - 2 / (e^(2 |x|) + 1), whose 1 no longer cancels.
__device__ __forceinline__ float tree_tanh(float x) {
    const float z = x * x, t = fabsf(x);
    const float small = x * fmaf(z, fmaf(z, 21.f, 1260.f), 10395.f) /
                        fmaf(z, fmaf(z, z + 210.f, 4725.f), 10395.f);
    const float e = __builtin_amdgcn_exp2f(2.8853900817779268f * t);
    const float big = copysignf(1.f - 2.f / (e + 1.f), x);
    return t <= 1.f ? small : big;
}

// Reductions over a wave, left in every lane.
template <bool MAX>
__device__ __forceinline__ float tree_wave_reduce(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(v, d, 64);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    return v;
}

constexpr int kTreeWaves = 4;

__global__ __launch_bounds__(kTreeWaves * 64) void tree_rows_kernel(TreeArgs a) {
    __shared__ float s_q[kTreeWaves][kHeadDim];
    __shared__ float s_p[kTreeWaves][64];
    __shared__ int s_off[kTreeWaves][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = blockIdx.x * kTreeWaves + wave;
    const bool live = row < a.n_tokens * a.Hq;
    const int t = live ? row / a.Hq : 0, h = live ? row - t * a.Hq : 0, kvh = h / a.G;
    // the token's sequence: the first b with q_indptr[b + 1] > t
    int b = t;
    if (a.q_indptr) {
        int lo = 0, hi = a.B;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.q_indptr[mid + 1] > t) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
    }
    if (!live || b >= a.B) return;   // (no barrier below: a wave keeps to its own LDS)
    const int q0 = a.q_indptr ? a.q_indptr[b] : b, n = a.q_indptr ? a.q_indptr[b + 1] - q0 : 1, i = t - q0;
    if (i < 0) return;
    const int pb = a.kv_indptr[b], np = a.kv_indptr[b + 1] - pb;
    const int len = np > 0 ? (np - 1) * kPage + min(kPage, max(1, a.kv_last[b])) : 0, ctx = len - n;
    const int pos_q = a.depth ? max(0, a.depth[t]) : i;   // relative to ctx, as below
    const float slope = a.slopes ? a.slopes[h] * 1.4426950408889634f : 0.f;
    const _Float16* q = a.q + ((size_t)t * a.Hq + h) * kHeadDim;
    s_q[wave][lane] = (float)q[lane];
    s_q[wave][lane + 64] = (float)q[lane + 64];
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int base = 0; base < len; base += 64) {
        const int key = base + lane, j = key - ctx;
        bool seen = key < len;
        int pos_k = j;
        if (seen && j >= 0) {
            if (a.mask || a.depth) seen = j < kTreeMaxTokens;
            if (seen) seen = a.mask ? j < 32 * a.mask_words && (a.mask[(size_t)t * a.mask_words + j / 32] >> (j & 31) & 1) : j <= i;
            if (seen && a.depth) pos_k = max(0, a.depth[q0 + j]);
        }
        if (a.window > 0 && seen) seen = pos_q - pos_k < a.window || key < a.sink;
        float x = -INFINITY;
        if (seen) {
            const size_t off = ((size_t)(uint32_t)a.kv_indices[pb + key / kPage] * kPage + key % kPage) * a.Hkv + kvh;
            const _Float16* k = reinterpret_cast<const _Float16*>(a.k) + off * kHeadDim;
            float dot = 0.f;
            for (int d = 0; d < kHeadDim; ++d) dot = fmaf(s_q[wave][d], (float)k[d], dot);
            x = a.cap_out > 0.f ? a.cap_out * tree_tanh(dot * a.cap_in) : dot * a.scale_log2;
            if (a.slopes) x = fmaf(slope, (float)(pos_k - pos_q), x);
        }
        const float mn = fmaxf(m, tree_wave_reduce<true>(x));
        const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float p = seen ? __builtin_amdgcn_exp2f(x - (mn == -INFINITY ? 0.f : mn)) : 0.f;
        m = mn;
        l = l * al + p;
        o0 *= al;
        o1 *= al;
        s_p[wave][lane] = p;
        s_off[wave][lane] = seen;
        __builtin_amdgcn_wave_barrier();
        for (int e = 0; e < 64; ++e) {
            if (!__builtin_amdgcn_readfirstlane(s_off[wave][e])) continue;
            const int k2 = base + e;
            const size_t off = ((size_t)(uint32_t)a.kv_indices[pb + k2 / kPage] * kPage + k2 % kPage) * a.Hkv + kvh;
            const _Float16* v = reinterpret_cast<const _Float16*>(a.v) + off * kHeadDim + 2 * lane;
            o0 = fmaf(s_p[wave][e], (float)v[0], o0);
            o1 = fmaf(s_p[wave][e], (float)v[1], o1);
        }
        __builtin_amdgcn_wave_barrier();
    }
    const float L = tree_wave_reduce<false>(l);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    _Float16* out = a.out + ((size_t)t * a.Hq + h) * kHeadDim + 2 * lane;
    out[0] = (_Float16)(o0 * inv);
    out[1] = (_Float16)(o1 * inv);
    if (lane == 0)
        a.lse[(size_t)t * a.Hq + h] = L == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(L)) * kTreeLn2;
}

}  // namespace

hipError_t launch_tree_attention(const TreeArgs& a, hipStream_t s) {
    const int64_t rows = (int64_t)a.n_tokens * a.Hq;
    if (rows <= 0 || a.B <= 0) return hipSuccess;
    tree_rows_kernel<<<(unsigned)((rows + kTreeWaves - 1) / kTreeWaves), kTreeWaves * 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace pdattn
