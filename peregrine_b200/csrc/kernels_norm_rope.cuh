// Query/key norms per head, rotation and the store into the cache, one pass over the projection's rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos * theta^(-2j/R)
//
// Every value is read once (4 bytes) and written once (2 bytes), so HBM bounds it.  A head is spread over
// D / 8 lanes of 8 values (two 16-byte loads each), which are whole pairs in both pairings, so neither the norm's
// sum nor the rotation leaves the warp.  The angles of a row are the same for all its heads: a CTA takes one
// row (or, when there are too few rows to fill the device, some heads of one) and computes its cosines once.
// Angles are formed and reduced to half turns in 64 bits: at position 10^6 an fp32 product is off by 0.03.
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
};

constexpr int kNrWarps = 8;

template <int D, bool BF16>
__global__ void __launch_bounds__(kNrWarps * 32) norm_rope_kernel(const NormRopeArgs P) {
    constexpr int LPH = D / 8;     // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads a warp works on at once
    __shared__ float s_cs[D / 2], s_sn[D / 2];
    const int row = blockIdx.x, seq = row / P.rows_per_seq;
    const int base = P.base[seq];
    if (base < 0) return;
    const int pos = P.pos[row], half = P.R >> 1;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        const double inv = exp2(-2.0 * j / P.R * log2((double)P.theta));
        double turns = (double)pos * inv * 0.15915494309189533577;
        turns -= rint(turns);
        sincospif((float)(2.0 * turns), &s_sn[j], &s_cs[j]);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / LPH, l = lane % LPH;
    const int heads = P.H + 2 * P.kv.n_kv;
    const long long slot = (long long)base + row % P.rows_per_seq;
    const float *x = P.qkv + (long long)row * P.row_stride;
    // 16-byte accesses of either pairing need the rotated part to end on a lane's boundary
    const bool wide = (P.R & 7) == 0;
    for (int h0 = (blockIdx.y * kNrWarps + warp) * HPW; h0 < heads; h0 += gridDim.y * kNrWarps * HPW) {
        const int h = h0 + sub;
        const bool there = h < heads;
        const int hx = there ? h : heads - 1;
        const bool is_q = hx < P.H, is_v = hx >= P.H + P.kv.n_kv;
        // Pair p of the head (4 of them to a lane): elements i0(p), i1(p) in, o0(p), o1(p) out.
        const bool turned = !is_v;
        const float *xh = x + (long long)hx * D;
        float a[4], b[4];
        int i0[4], i1[4];
        const int p0 = 4 * l;
        const bool style1 = P.style == 1 && turned && p0 < half;
        if (wide) {
            if (style1) {
                const float4 u = *reinterpret_cast<const float4 *>(xh + p0), w = *reinterpret_cast<const float4 *>(xh + half + p0);
                a[0] = u.x, a[1] = u.y, a[2] = u.z, a[3] = u.w;
                b[0] = w.x, b[1] = w.y, b[2] = w.z, b[3] = w.w;
            } else {
                const float4 u = *reinterpret_cast<const float4 *>(xh + 2 * p0), w = *reinterpret_cast<const float4 *>(xh + 2 * p0 + 4);
                a[0] = u.x, b[0] = u.y, a[1] = u.z, b[1] = u.w;
                a[2] = w.x, b[2] = w.y, a[3] = w.z, b[3] = w.w;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int p = p0 + e;
            const bool halves = P.style == 1 && turned && p < half;
            i0[e] = halves ? p : 2 * p;
            i1[e] = halves ? half + p : 2 * p + 1;
            if (!wide) {
                a[e] = xh[i0[e]];
                b[e] = xh[i1[e]];
            }
        }
        const float *w = is_v ? nullptr : is_q ? P.q_w : P.k_w;
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w) {
            const float r = __frsqrt_rn(ss * (1.0f / D) + P.eps);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = a[e] * r * __ldg(w + i0[e]);
                b[e] = b[e] * r * __ldg(w + i1[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (turned && p0 + e < half) {
                const float cs = s_cs[p0 + e], sn = s_sn[p0 + e], u = a[e], v = b[e];
                a[e] = u * cs - v * sn;
                b[e] = v * cs + u * sn;
            }
        if (!there) continue;
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
            if (turned && p0 < half) {
                *reinterpret_cast<uint2 *>(out + p0) = make_uint2(pack16<BF16>(a[0], a[1]), pack16<BF16>(a[2], a[3]));
                *reinterpret_cast<uint2 *>(out + half + p0) = make_uint2(pack16<BF16>(b[0], b[1]), pack16<BF16>(b[2], b[3]));
            } else {
                *reinterpret_cast<uint4 *>(out + 2 * p0) = make_uint4(pack16<BF16>(a[0], b[0]), pack16<BF16>(a[1], b[1]),
                                                                      pack16<BF16>(a[2], b[2]), pack16<BF16>(a[3], b[3]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = p0 + e;
                const bool t = turned && p < half;
                const uint32_t both = pack16<BF16>(a[e], b[e]);
                out[t ? p : 2 * p] = (uint16_t)both;
                out[t ? half + p : 2 * p + 1] = (uint16_t)(both >> 16);
            }
        }
    }
}

}  // namespace pgb
