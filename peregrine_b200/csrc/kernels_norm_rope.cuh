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
// Measured: 4096 rows of 48 + 16 heads of 128 in 38 us, 5.3 TB/s (81 % of the copy rate).  A warp's instructions count as much
// as HBM: with 186 of them for its 256 values the same took 43.5 us; two operations of the norm to an instruction, places that
// grow with the heads and kernels of their own for unaligned rotations took off the rest.
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

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// WIDE: the rotated part ends on a lane's boundary (R a multiple of 8), so a lane's values are two pieces of 16 bytes.
template <int D, bool BF16, bool WIDE>
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
    const int first = (int)(items * w / warps), count = (int)(items * (w + 1) / warps) - first;
    float *buf = nr_smem + warp * 2 * kNrSteps * 256;
    int row = first / P.parts, part = first - row * P.parts;  // of the item being worked on
    int to_row = row, to_part = part;                         // of the item to bring next
    auto fetch = [&](int at) {                                // into half `at` of the buffer
        const int h0 = to_part * P.per * HPW, n = min(P.per * HPW, heads - h0);
        if (lane == 0) {
            mbar_expect_tx(bar + 8 * at, (uint32_t)(n * D * 4));
            bulk_g2s(smem_u32(buf + at * kNrSteps * 256), P.qkv + (long long)to_row * P.row_stride + (long long)h0 * D, (uint32_t)(n * D * 4), bar + 8 * at);
        }
        if (++to_part == P.parts) {
            to_part = 0;
            ++to_row;
        }
    };
    for (int j = threadIdx.x; j < half; j += blockDim.x)  // turns per position
        s_freq[j] = exp2(-2.0 * j / P.R * P.log2_theta) * 0.15915494309189533577;
    griddep_wait();
    griddep_launch_dependents();
    if (count > 0) fetch(0);
    const int sub = lane / LPH, l = lane % LPH, p0 = 4 * l;  // this lane's pairs of a head: p0 .. p0 + 3
    const bool turned = p0 < half, halves = P.style == 1;    // pairs (j, R / 2 + j) instead of (2j, 2j + 1)
    // where pair p of a head stands (not rotated: 2p, 2p + 1)
    auto one = [&](int p) { return halves && p < half ? p : 2 * p; };
    auto two = [&](int p) { return halves && p < half ? half + p : 2 * p + 1; };
    // WIDE: this lane's two pieces of a head, [in0, + 4) and [in1, + 4); where a rotated head's go
    const int in0 = halves && turned ? p0 : 2 * p0, in1 = halves && turned ? half + p0 : 2 * p0 + 4;
    // the weights of the kind of head (0 query, 1 key, 2 value) that this lane works on; kinds follow one another
    float wt[8];
    int kind = -1;
    auto weights = [&](int to) {
        kind = to;
        const float *w = to == 0 ? P.q_w : P.k_w;
        if (to == 2 || !w) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            wt[e] = w[WIDE ? in0 + e : one(p0 + e)];
            wt[4 + e] = w[WIDE ? in1 + e : two(p0 + e)];
        }
    };
    float cs[4], sn[4];
    int base = 0, pos = 0, seq = 0;
    long long slot = 0, kv_row = 0;  // of the row; its first element in the cache
    uint16_t *q_row = nullptr;
    if (count > 0) {
        seq = row / P.rows_per_seq;
        base = P.base[seq];
        pos = P.pos[row];
    }
    __syncthreads();
    bool fresh = true;
    for (int item = 0; item < count; ++item) {
        if (item + 1 < count) fetch((item + 1) & 1);
        if (fresh) {
            if (item) {
                seq = row / P.rows_per_seq;
                base = P.base[seq];
                pos = P.pos[row];
            }
            slot = (long long)base + (row - seq * P.rows_per_seq);
            kv_row = (long long)seq * P.kv.seq_stride + slot * P.kv.slot_stride;
            q_row = P.q_out + (long long)row * P.H * D;
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
        um_spin(bar + 8 * (item & 1), (uint32_t)((item >> 1) & 1), fail);
        const float *x = buf + (item & 1) * kNrSteps * 256 + sub * D;
        const int step0 = part * P.per, steps = base < 0 ? 0 : min(P.per, P.steps - step0);
        int h = step0 * HPW + sub;
        for (int s = 0; s < steps; ++s, h += HPW, x += HPW * D) {
            const int is = h < P.H ? 0 : h < P.H + P.kv.n_kv ? 1 : 2;
            float a[4], b[4];  // (past the last head: what the buffer held before, and not used)
            if (WIDE) {
                const float4 v = *reinterpret_cast<const float4 *>(x + in0), u = *reinterpret_cast<const float4 *>(x + in1);
                a[0] = v.x, a[1] = v.y, a[2] = v.z, a[3] = v.w;
                b[0] = u.x, b[1] = u.y, b[2] = u.z, b[3] = u.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] = x[is == 2 ? 2 * (p0 + e) : one(p0 + e)];
                    b[e] = x[is == 2 ? 2 * (p0 + e) + 1 : two(p0 + e)];
                }
            }
            float2 sq = mul2(make_float2(a[0], a[1]), make_float2(a[0], a[1]));
            sq = fma2(make_float2(a[2], a[3]), make_float2(a[2], a[3]), sq);
            sq = fma2(make_float2(b[0], b[1]), make_float2(b[0], b[1]), sq);
            sq = fma2(make_float2(b[2], b[3]), make_float2(b[2], b[3]), sq);
            float ss = sq.x + sq.y;
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (h >= heads) continue;
            if (is != kind) weights(is);
            uint16_t *out;
            if (is == 0) {
                out = q_row + h * D;
            } else {
                if (slot >= P.kv.cap) continue;
                const int kvh = h - P.H - (is == 2 ? P.kv.n_kv : 0);
                out = (is == 2 ? P.kv.v : P.kv.k) + kv_row + kvh * P.kv.head_stride;
                if (is == 1 && l == 0) {
                    const long long to = ((long long)seq * P.kv.n_kv + kvh) * P.kv.cap + slot;
                    if (P.kv.pos) P.kv.pos[to] = pos;
                    if (P.kv.acc) P.kv.acc[to] = 0.0f;
                }
            }
            if (is == 0 ? P.q_w != nullptr : is == 1 && P.k_w != nullptr) {
                const float rs = rsqrtf(fmaf(ss, 1.0f / D, P.eps));
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float2 r2 = make_float2(rs, rs);
                    const float2 y = mul2(make_float2(a[e], a[e + 1]), mul2(r2, make_float2(wt[e], wt[e + 1])));
                    const float2 z = mul2(make_float2(b[e], b[e + 1]), mul2(r2, make_float2(wt[4 + e], wt[5 + e])));
                    a[e] = y.x, a[e + 1] = y.y;
                    b[e] = z.x, b[e + 1] = z.y;
                }
            }
            if (WIDE) {
                uint32_t p[4];
                if (!halves && turned && is != 2) {  // pairs stand side by side, and part
                    float c[4], d[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = e < 2 ? a[2 * e] : b[2 * e - 4], u = e < 2 ? a[2 * e + 1] : b[2 * e - 3];
                        c[e] = fmaf(v, cs[e], -(u * sn[e]));
                        d[e] = fmaf(u, cs[e], v * sn[e]);
                    }
                    p[0] = pack16<BF16>(c[0], c[1]), p[1] = pack16<BF16>(c[2], c[3]);
                    p[2] = pack16<BF16>(d[0], d[1]), p[3] = pack16<BF16>(d[2], d[3]);
                } else {
                    if (halves && turned && is != 2) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = a[e], u = b[e];
                            a[e] = fmaf(v, cs[e], -(u * sn[e]));
                            b[e] = fmaf(u, cs[e], v * sn[e]);
                        }
                    }
                    p[0] = pack16<BF16>(a[0], a[1]), p[1] = pack16<BF16>(a[2], a[3]);
                    p[2] = pack16<BF16>(b[0], b[1]), p[3] = pack16<BF16>(b[2], b[3]);
                }
                if (turned && (halves || is != 2)) {
                    *reinterpret_cast<uint2 *>(out + p0) = make_uint2(p[0], p[1]);
                    *reinterpret_cast<uint2 *>(out + half + p0) = make_uint2(p[2], p[3]);
                } else {
                    *reinterpret_cast<uint4 *>(out + 2 * p0) = make_uint4(p[0], p[1], p[2], p[3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int p = p0 + e;
                    const bool t = is != 2 && p < half;
                    if (t) {
                        const float v = a[e], u = b[e];
                        a[e] = fmaf(v, cs[e], -(u * sn[e]));
                        b[e] = fmaf(u, cs[e], v * sn[e]);
                    }
                    const uint32_t both = pack16<BF16>(a[e], b[e]);
                    out[t ? p : 2 * p] = (uint16_t)both;
                    out[t ? half + p : 2 * p + 1] = (uint16_t)(both >> 16);
                }
            }
        }
        if (++part == P.parts) {
            part = 0;
            ++row;
            fresh = true;
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
