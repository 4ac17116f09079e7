// Query/key norms per head, rotation and the store into the cache, one pass over the projection's rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos * theta^(-2j/R)
//
// Every value is read once (4 bytes) and written once (2 bytes), so HBM bounds it.  A head is spread over
// D / 8 lanes of 8 values (two 16-byte loads each), which are whole pairs in both pairings, so neither the norm's
// sum nor the rotation leaves the warp, and a warp takes 256 / D heads at a time.  What a lane needs of the weights and of a
// row's cosines is the same for all heads of the row: a warp works on a run of heads of one row and keeps both in
// registers, with the loads of four steps under way.  Frequencies (64 bits) are formed once per CTA.
// Angles are formed and reduced to turns in 64 bits: at position 10^6 an fp32 product is off by 0.03.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace pgb {

// A cache as the kernels see it (ColiCudaKv with its strides filled in).
struct KvArgs {
    uint16_t *k, *v;
    int32_t *pos;
    float *acc;
    int n_seq, n_kv, cap, D;
    long long seq_stride, head_stride, slot_stride;
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {  // a in the low half, both to nearest even
    uint32_t r;
    if (BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

struct NormRopeArgs {
    uint16_t *q_out;
    const float *qkv;
    long long row_stride;
    int H;
    KvArgs kv;
    const float *q_w, *k_w;
    float eps;
    const int *pos, *base;
    int rows_per_seq;
    float theta;
    int R, style;
    int rows, steps, per, parts;  // rows, steps (256 / D heads) of a row, of an item; items of a row
};

constexpr int kNrWarps = 8;

template <int D, bool BF16>
__global__ void __launch_bounds__(kNrWarps * 32, 2) norm_rope_kernel(const NormRopeArgs P) {
    constexpr int LPH = D / 8;     // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads of a step
    constexpr int U = 4;           // steps whose loads are under way together
    __shared__ double s_freq[D / 2];
    const int half = P.R >> 1;
    for (int j = threadIdx.x; j < half; j += blockDim.x)  // turns per position
        s_freq[j] = exp2(-2.0 * j / P.R * log2((double)P.theta)) * 0.15915494309189533577;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / LPH, l = lane % LPH, p0 = 4 * l;  // this lane's pairs of a head: p0 .. p0 + 3
    const int heads = P.H + 2 * P.kv.n_kv;
    // 16-byte accesses of either pairing need the rotated part to end on a lane's boundary
    const bool wide = (P.R & 7) == 0, turned = p0 < half;
    // elements of pair p of a rotated head, in and out (values and what is not rotated: 2p, 2p + 1)
    auto first = [&](int p) { return P.style == 1 && p < half ? p : 2 * p; };
    auto second = [&](int p) { return P.style == 1 && p < half ? half + p : 2 * p + 1; };
    float wq[8], wk[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        wq[e] = P.q_w ? P.q_w[first(p0 + e)] : 1.0f;
        wq[4 + e] = P.q_w ? P.q_w[second(p0 + e)] : 1.0f;
        wk[e] = P.k_w ? P.k_w[first(p0 + e)] : 1.0f;
        wk[4 + e] = P.k_w ? P.k_w[second(p0 + e)] : 1.0f;
    }
    const int items = P.rows * P.parts;
    for (int item = blockIdx.x * kNrWarps + warp; item < items; item += gridDim.x * kNrWarps) {
        const int row = item / P.parts, seq = row / P.rows_per_seq, step0 = (item - row * P.parts) * P.per;
        const int base = P.base[seq], pos = P.pos[row];
        if (base < 0) continue;
        const long long slot = (long long)base + (row - seq * P.rows_per_seq);
        const float *x = P.qkv + (long long)row * P.row_stride;
        float cs[4], sn[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            cs[e] = 1.0f, sn[e] = 0.0f;
            if (p0 + e < half) {
                double t = (double)pos * s_freq[p0 + e];
                t -= rint(t);
                sincospif((float)(2.0 * t), &sn[e], &cs[e]);
            }
        }
        const int end = min(step0 + P.per, P.steps);
        for (int s0 = step0; s0 < end; s0 += U) {
            float a[U][4], b[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = (s0 + u) * HPW + sub;
                if (s0 + u >= end || h >= heads) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[u][e] = b[u][e] = 0.0f;
                    continue;
                }
                const float *xh = x + (long long)h * D;
                const bool halves = P.style == 1 && h < P.H + P.kv.n_kv;
                if (wide) {
                    const bool split = halves && turned;
                    const float4 v = __ldcs(reinterpret_cast<const float4 *>(xh + (split ? p0 : 2 * p0)));
                    const float4 w = __ldcs(reinterpret_cast<const float4 *>(xh + (split ? half + p0 : 2 * p0 + 4)));
                    if (split) {
                        a[u][0] = v.x, a[u][1] = v.y, a[u][2] = v.z, a[u][3] = v.w;
                        b[u][0] = w.x, b[u][1] = w.y, b[u][2] = w.z, b[u][3] = w.w;
                    } else {
                        a[u][0] = v.x, b[u][0] = v.y, a[u][1] = v.z, b[u][1] = v.w;
                        a[u][2] = w.x, b[u][2] = w.y, a[u][3] = w.z, b[u][3] = w.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[u][e] = xh[halves ? first(p0 + e) : 2 * (p0 + e)];
                        b[u][e] = xh[halves ? second(p0 + e) : 2 * (p0 + e) + 1];
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = (s0 + u) * HPW + sub;
                const bool is_q = h < P.H, is_v = h >= P.H + P.kv.n_kv;
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fmaf(a[u][e], a[u][e], fmaf(b[u][e], b[u][e], ss));
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (s0 + u >= end || h >= heads) continue;
                if (!is_v) {
                    if (is_q ? P.q_w != nullptr : P.k_w != nullptr) {
                        const float r = __frsqrt_rn(ss * (1.0f / D) + P.eps);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            a[u][e] = a[u][e] * r * (is_q ? wq[e] : wk[e]);
                            b[u][e] = b[u][e] * r * (is_q ? wq[4 + e] : wk[4 + e]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {  // (not rotated: cosine 1, sine 0; infinities must not become 0 x inf)
                        const float v = a[u][e], w = b[u][e];
                        if (p0 + e < half) {
                            a[u][e] = v * cs[e] - w * sn[e];
                            b[u][e] = w * cs[e] + v * sn[e];
                        }
                    }
                }
                uint16_t *out;
                if (is_q) {
                    out = P.q_out + ((long long)row * P.H + h) * D;
                } else {
                    if (slot >= P.kv.cap) continue;
                    const int kvh = is_v ? h - P.H - P.kv.n_kv : h - P.H;
                    out = (is_v ? P.kv.v : P.kv.k) + (long long)seq * P.kv.seq_stride + kvh * P.kv.head_stride + slot * P.kv.slot_stride;
                    if (!is_v && l == 0) {
                        const long long at = ((long long)seq * P.kv.n_kv + kvh) * P.kv.cap + slot;
                        if (P.kv.pos) P.kv.pos[at] = pos;
                        if (P.kv.acc) P.kv.acc[at] = 0.0f;
                    }
                }
                if (wide) {
                    if (!is_v && turned) {
                        *reinterpret_cast<uint2 *>(out + p0) = make_uint2(pack16<BF16>(a[u][0], a[u][1]), pack16<BF16>(a[u][2], a[u][3]));
                        *reinterpret_cast<uint2 *>(out + half + p0) = make_uint2(pack16<BF16>(b[u][0], b[u][1]), pack16<BF16>(b[u][2], b[u][3]));
                    } else {
                        *reinterpret_cast<uint4 *>(out + 2 * p0) = make_uint4(pack16<BF16>(a[u][0], b[u][0]), pack16<BF16>(a[u][1], b[u][1]),
                                                                              pack16<BF16>(a[u][2], b[u][2]), pack16<BF16>(a[u][3], b[u][3]));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int p = p0 + e;
                        const bool t = !is_v && p < half;
                        const uint32_t both = pack16<BF16>(a[u][e], b[u][e]);
                        out[t ? p : 2 * p] = (uint16_t)both;
                        out[t ? half + p : 2 * p + 1] = (uint16_t)(both >> 16);
                    }
                }
            }
        }
    }
}

}  // namespace pgb
