// Query/key norms per head, rotation and the store into the cache, one pass over the projection's rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = pos * theta^(-2j/R)
//
// Every value is read once (4 bytes) and written once (2 bytes), so HBM bounds it.  A head is spread over
// D / 8 lanes of 8 values (two 16-byte loads each), which are whole pairs in both pairings, so neither the norm's
// sum nor the rotation leaves the warp, and a warp takes 256 / D heads at a time.  What a lane needs of the weights and of a
// row's cosines is the same for all heads of the row: a warp works on a stretch of the batch's heads in order and keeps both in
// registers; its input comes by bulk copies of up to 4 kB, one being worked on and one under way (24 warps an SM, 96 kB).
// Frequencies (64 bits) are formed once per CTA.
// Measured: 4096 rows of 48 + 16 heads of 128 in 43 us, 4.7 TB/s (72 % of the copy rate); about 150 instructions for a warp's
// 256 values keep the issue slots as busy as HBM.
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
    double log2_theta;
    int R, style;
    int rows, steps, per, parts;  // rows, steps (256 / D heads) of a row, of an item; items of a row
    int *err;
};

constexpr int kNrWarps = 8, kNrSteps = 4, kNrPerSm = 3;  // warps of a CTA, most steps (1 kB) of an item, CTAs of an SM
constexpr int kNrSmem = kNrWarps * 2 * kNrSteps * 1024;

template <int D, bool BF16>
__global__ void __launch_bounds__(kNrWarps * 32, kNrPerSm) norm_rope_kernel(const NormRopeArgs P) {
    constexpr int LPH = D / 8;     // lanes of a head
    constexpr int HPW = 32 / LPH;  // heads of a step
    extern __shared__ __align__(128) float nr_smem[];
    __shared__ double s_freq[D / 2];
    __shared__ __align__(8) unsigned long long s_bar[kNrWarps][2];
    __shared__ int s_fail;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = P.R >> 1;
    const int heads = P.H + 2 * P.kv.n_kv;
    const uint32_t bar = smem_u32(&s_bar[warp][0]);
    if (lane == 0) {
        mbar_init(bar, 1);
        mbar_init(bar + 8, 1);
        fence_mbar_init();
        if (warp == 0) s_fail = 0;
    }
    __syncwarp();
    volatile int *fail = &s_fail;
    // this warp's stretch of items, `per` steps of a row each
    const long long items = (long long)P.rows * P.parts, warps = (long long)gridDim.x * kNrWarps, w = (long long)blockIdx.x * kNrWarps + warp;
    const int first = (int)(items * w / warps), end = (int)(items * (w + 1) / warps);
    float *buf = nr_smem + warp * 2 * kNrSteps * 256;
    auto fetch = [&](int item) {  // into the half of the buffer that its number says
        const int row = item / P.parts, h0 = (item - row * P.parts) * P.per * HPW, n = min(P.per * HPW, heads - h0);
        const int at = (item - first) & 1;
        if (lane == 0) {
            mbar_expect_tx(bar + 8 * at, (uint32_t)(n * D * 4));
            bulk_g2s(smem_u32(buf + at * kNrSteps * 256), P.qkv + (long long)row * P.row_stride + (long long)h0 * D, (uint32_t)(n * D * 4), bar + 8 * at);
        }
    };
    for (int j = threadIdx.x; j < half; j += blockDim.x)  // turns per position
        s_freq[j] = exp2(-2.0 * j / P.R * P.log2_theta) * 0.15915494309189533577;
    griddep_wait();
    griddep_launch_dependents();
    if (first < end) fetch(first);
    const int sub = lane / LPH, l = lane % LPH, p0 = 4 * l;  // this lane's pairs of a head: p0 .. p0 + 3
    // 16-byte accesses of either pairing need the rotated part to end on a lane's boundary
    const bool wide = (P.R & 7) == 0, turned = p0 < half;
    // elements of pair p of a rotated head (values and what is not rotated: 2p, 2p + 1)
    auto one = [&](int p) { return P.style == 1 && p < half ? p : 2 * p; };
    auto two = [&](int p) { return P.style == 1 && p < half ? half + p : 2 * p + 1; };
    // the weights of the kind of head (0 query, 1 key, 2 value) that this lane works on; kinds follow one another
    float wt[8];
    int kind = -1;
    auto weights = [&](int to) {
        kind = to;
        const float *w = to == 0 ? P.q_w : P.k_w;
        if (to == 2 || !w) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            wt[e] = w[one(p0 + e)];
            wt[4 + e] = w[two(p0 + e)];
        }
    };
    float cs[4], sn[4];
    int row = -1, base = 0, pos = 0;
    if (first < end) {
        row = first / P.parts;
        base = P.base[row / P.rows_per_seq];
        pos = P.pos[row];
    }
    __syncthreads();
    bool fresh = true;
    for (int item = first; item < end; ++item) {
        if (item + 1 < end) fetch(item + 1);
        const int r = item / P.parts, step0 = (item - r * P.parts) * P.per;
        if (r != row || fresh) {
            if (!fresh) {
                row = r;
                base = P.base[row / P.rows_per_seq];
                pos = P.pos[row];
            }
            fresh = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                cs[e] = 1.0f, sn[e] = 0.0f;
                if (p0 + e < half) {
                    double t = (double)pos * s_freq[p0 + e];
                    t -= rint(t);
                    sincospif((float)(2.0 * t), &sn[e], &cs[e]);
                }
            }
        }
        const int at = (item - first) & 1, seq = row / P.rows_per_seq;
        um_spin(bar + 8 * at, (uint32_t)(((item - first) >> 1) & 1), fail);
        const long long slot = (long long)base + (row - seq * P.rows_per_seq);
        const float *x = buf + at * kNrSteps * 256;
        const int steps = base < 0 ? 0 : min(P.per, P.steps - step0);
        for (int s = 0; s < steps; ++s) {
            const int h = (step0 + s) * HPW + sub;
            const bool there = h < heads, is_q = h < P.H, is_v = h >= P.H + P.kv.n_kv;
            const float *xh = x + (s * HPW + (there ? sub : 0)) * D;
            float a[4], b[4];
            if (wide) {
                const bool split = P.style == 1 && !is_v && turned;
                const float4 v = *reinterpret_cast<const float4 *>(xh + (split ? p0 : 2 * p0));
                const float4 u = *reinterpret_cast<const float4 *>(xh + (split ? half + p0 : 2 * p0 + 4));
                if (split) {
                    a[0] = v.x, a[1] = v.y, a[2] = v.z, a[3] = v.w;
                    b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w;
                } else {
                    a[0] = v.x, b[0] = v.y, a[1] = v.z, b[1] = v.w;
                    a[2] = u.x, b[2] = u.y, a[3] = u.z, b[3] = u.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] = xh[is_v ? 2 * (p0 + e) : one(p0 + e)];
                    b[e] = xh[is_v ? 2 * (p0 + e) + 1 : two(p0 + e)];
                }
            }
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (!there) continue;
            const int is = is_q ? 0 : is_v ? 2 : 1;
            if (is != kind) weights(is);
            if (!is_v) {
                if (is_q ? P.q_w != nullptr : P.k_w != nullptr) {
                    const float rs = __frsqrt_rn(fmaf(ss, 1.0f / D, P.eps));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] *= rs * wt[e];
                        b[e] *= rs * wt[4 + e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (p0 + e < half) {
                        const float v = a[e], u = b[e];
                        a[e] = fmaf(v, cs[e], -(u * sn[e]));
                        b[e] = fmaf(u, cs[e], v * sn[e]);
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
                    const long long to = ((long long)seq * P.kv.n_kv + kvh) * P.kv.cap + slot;
                    if (P.kv.pos) P.kv.pos[to] = pos;
                    if (P.kv.acc) P.kv.acc[to] = 0.0f;
                }
            }
            if (wide) {
                if (!is_v && turned) {
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
                    const bool t = !is_v && p < half;
                    const uint32_t both = pack16<BF16>(a[e], b[e]);
                    out[t ? p : 2 * p] = (uint16_t)both;
                    out[t ? half + p : 2 * p + 1] = (uint16_t)(both >> 16);
                }
            }
        }
        __syncwarp();  // all have read this half of the buffer before the copy after next fills it
    }
    if (lane == 0 && *fail) {
        report_error(P.err, kErrBarrierTimeout);
        const long long t0 = clock64();  // copies that are under way land before the shared memory is given back
        while (clock64() - t0 < 4000000LL) {
        }
    }
}

}  // namespace pgb
