// Attention of a batch behind a shared prefix: out = softmax(scale q.k) v, one row and head per CTA.
#pragma once
#include "kernels_norm_rope.cuh"

namespace pgb {

struct AttnArgs {
    void *out;
    int out_f32;
    const uint16_t *q;
    int S, H, G;  // rows, query heads, query heads per kv head
    KvArgs pre, own;
    int prefix_len;
    const int *base;
    int rows;
    const unsigned long long *mask;
    float scale;
    float *stats;  // [S, H] pairs: maximum of the scaled scores, 1 / sum (0: the row sees nothing)
};

template <bool BF16>
__device__ __forceinline__ float from16(uint16_t v) {
    return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// Own slots that row `i` of a sequence may see: t < base, and new slots by mask or order.
__device__ __forceinline__ bool sees(int t, int base, int i, unsigned long long mask) {
    return t < base || ((mask >> (t - base)) & 1ull);
}
__device__ __forceinline__ unsigned long long row_mask(const AttnArgs &P, int row, int i) {
    const unsigned long long in = P.rows == 64 ? ~0ull : (1ull << P.rows) - 1;
    return (P.mask ? P.mask[row] : ~0ull >> (63 - i)) & in;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(128) attn_rows_kernel(const AttnArgs P) {
    constexpr int E = D / 32;
    const int row = blockIdx.x / P.H, h = blockIdx.x % P.H, seq = row / P.rows, i = row % P.rows, kvh = h / P.G;
    const int base = P.base[seq];
    if (base < 0) return;
    const unsigned long long mask = row_mask(P, row, i);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n_own = (int)min((long long)base + P.rows, (long long)P.own.cap);
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) {
        q[e] = from16<BF16>(P.q[((long long)row * P.H + h) * D + lane * E + e]);
        o[e] = 0.0f;
    }
    const long long total = (long long)P.prefix_len + n_own;
    for (long long t = warp; t < total; t += 4) {
        const bool own = t >= P.prefix_len;
        const KvArgs &kv = own ? P.own : P.pre;
        const int slot = (int)(own ? t - P.prefix_len : t);
        if (own && !sees(slot, base, i, mask)) continue;
        const long long at = (own ? (long long)seq * kv.seq_stride : 0) + kvh * kv.head_stride + slot * kv.slot_stride + lane * E;
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s = fmaf(q[e], from16<BF16>(kv.k[at + e]), s);
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= P.scale;
        const float mn = fmaxf(m, s);
        if (mn == -INFINITY) continue;
        const float a = expf(m - mn), p = expf(s - mn);
        l = l * a + p;
        for (int e = 0; e < E; ++e) o[e] = o[e] * a + p * from16<BF16>(kv.v[at + e]);
        m = mn;
    }
    __shared__ float s_m[4], s_l[4], s_o[4][D];
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    __syncthreads();
    float mm = -INFINITY, ll = 0.0f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, s_m[w]);
    for (int w = 0; w < 4; ++w)
        if (s_l[w] != 0.0f) ll += s_l[w] * expf(s_m[w] - mm);
    for (int d = threadIdx.x; d < D; d += 128) {
        float v = 0.0f;
        for (int w = 0; w < 4; ++w)
            if (s_l[w] != 0.0f) v += s_o[w][d] * expf(s_m[w] - mm);
        if (ll != 0.0f) v /= ll;
        const long long at = ((long long)row * P.H + h) * D + d;
        if (P.out_f32)
            static_cast<float *>(P.out)[at] = v;
        else
            static_cast<uint16_t *>(P.out)[at] = (uint16_t)pack16<BF16>(v, 0.0f);
    }
    if (threadIdx.x == 0) {
        P.stats[((long long)row * P.H + h) * 2] = mm;
        P.stats[((long long)row * P.H + h) * 2 + 1] = ll != 0.0f ? 1.0f / ll : 0.0f;
    }
}

// acc[slot] += the weights that the rows and heads of its group gave it; one warp per slot.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attn_acc_kernel(const AttnArgs P) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int slot = (int)(w % P.own.cap);
    const long long g = w / P.own.cap;
    const int seq = (int)(g / P.own.n_kv), kvh = (int)(g % P.own.n_kv);
    if (seq >= P.own.n_seq) return;
    const int base = P.base[seq];
    if (base < 0 || slot >= (long long)base + P.rows) return;
    const long long at = (long long)seq * P.own.seq_stride + kvh * P.own.head_stride + slot * P.own.slot_stride + lane * E;
    float sum = 0.0f;
    for (int i = 0; i < P.rows; ++i) {
        const int row = seq * P.rows + i;
        if (!sees(slot, base, i, row_mask(P, row, i))) continue;
        for (int h = kvh * P.G; h < (kvh + 1) * P.G; ++h) {
            float s = 0.0f;
            for (int e = 0; e < E; ++e)
                s = fmaf(from16<BF16>(P.q[((long long)row * P.H + h) * D + lane * E + e]), from16<BF16>(P.own.k[at + e]), s);
            for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const float *st = P.stats + ((long long)row * P.H + h) * 2;
            if (st[1] != 0.0f) sum += expf(s * P.scale - st[0]) * st[1];
        }
    }
    if (lane == 0) P.own.acc[w] += sum;
}

}  // namespace pgb
