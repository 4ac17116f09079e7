// Attention of a batch behind a shared prefix: out = softmax(scale q.k) v.
//
// Problems: the prefix, once per kv head, with the rows of ALL sequences (its keys are read once for the batch), and every
// sequence's own slots per kv head with that sequence's rows.  A problem has M = rows x group query vectors, cut into
// row tiles of 16, 32 or 64.  Work is counted in tiles of 64 keys; all tiles of all problems form one line, and CTA c of
// n takes the c-th equal part of it, whatever the lengths (read on the device): no sequence is too long or too short.  Within its part
// a CTA keeps the running maximum m, sum l and output of one problem at a time (log2 units)
//     m' = max(m, x),  l' = l 2^(m-m') + sum 2^(x-m'),  o' = o 2^(m-m') + sum 2^(x-m') v,   x = scale log2(e) q.k
// and writes them as one partial result when the problem or the part ends.  A second launch joins the partials of a row in
// the order of the CTAs (no atomics) and adds up the weights that the slots received.
#pragma once
#include "kernels_norm_rope.cuh"

namespace pgb {

constexpr int kAtKeys = 64;      // keys of a tile
constexpr int kAtThreads = 128;  // 4 warps: row blocks of 16 x key ranges, by the row tile
constexpr int kAtCombine = 128;

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
    float scale2;                // scale * log2(e)
    int ctas;                    // CTAs that share the line of tiles
    int rt_pre, rt_own, rt_max;  // rows of a row tile: 16, 32 or 64
    int mt_pre, mt_own;          // row tiles of a problem (mt_pre 0: no prefix)
    // Tiles of tc_keys keys that every row of the problem sees, of problems with many rows, go to the tensor-memory
    // kernel (kernels_attn_tc.cuh); this one keeps what is left: the keys from cut_pre (prefix) or own_cut (own) on.
    int tc_keys;             // 64 or 128
    int tc_pre, tc_own;      // whether the prefix, the own slots are split this way
    int cut_pre;             // keys of the prefix that the tensor-memory kernel takes
    int tc_ctas, tc_rows;    // its CTAs, rows of one of its partials
    int tcm_pre, tcm_own;    // its row tiles of a problem
    int tc2_pre, tc2_own;    // 1: a row tile has 128 rows and its keys go to two halves of a partial in turn
    float *tc_part;          // [its problems x row tiles + tc_ctas][tc_rows][D]
    float2 *tc_ml;
    int *tc_offs;  // [n_seq + 1]: its tiles of the sequences before b
    int *err;
    // scratch
    float *part;    // [problems x row tiles + ctas][rt_max][D]: outputs of the partials, unnormalised
    float2 *ml;     // [..][rt_max]: their m and l
    int *offs;      // [n_seq + 1]: key tiles of the sequences before b
    float *scores;  // [n_seq][n_kv][rows * G][cap]: x of the own slots (-inf: not seen); only with acc
};

template <bool BF16>
__device__ __forceinline__ float from16(uint16_t v) {
    return BF16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Own slots in use by sequence b's call: all that its rows can see lie below.
__device__ __forceinline__ int own_keys(const AttnArgs &P, int b) {
    const int base = P.base[b];
    return base < 0 ? 0 : (int)min((long long)base + P.rows, (long long)P.own.cap);
}
// How many of them the tensor-memory kernel takes.
__device__ __forceinline__ int own_cut(const AttnArgs &P, int b) {
    if (!P.tc_own) return 0;
    const int base = P.base[b];
    return base < 0 ? 0 : min(base, P.own.cap) / P.tc_keys * P.tc_keys;
}
// New slots that row i of a sequence sees, a bit each.
__device__ __forceinline__ unsigned long long row_mask(const AttnArgs &P, int row, int i) {
    const unsigned long long in = P.rows == 64 ? ~0ull : (1ull << P.rows) - 1;
    return (P.mask ? P.mask[row] : ~0ull >> (63 - i)) & in;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {  // the rest of the 16 bytes is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Weights enter the second product in 16-bit terms.  A 16-bit output needs one (its own rounding is as large).  An fp32
// output takes as many as give it 22 bits: two of f16, three of bf16.  f16 weights are scaled by 2^10 so that their lower term
// stays a normal number down to weights of 2^-13 of the row's largest; l carries the same factor, so it cancels.
template <bool BF16>
constexpr float kAtLift = BF16 ? 0.0f : 10.0f;
template <bool BF16, bool F32>
constexpr int kAtTerms = F32 ? (BF16 ? 3 : 2) : 1;

template <bool BF16>
__device__ __forceinline__ float low16(uint32_t v) { return from16<BF16>((uint16_t)v); }
template <bool BF16>
__device__ __forceinline__ float high16(uint32_t v) { return from16<BF16>((uint16_t)(v >> 16)); }

// Two 16-bit values with zeros in the place of infinities and NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t finite16(uint32_t v) {
    constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
    return ((v & e) == e ? 0u : v & 0xFFFFu) | (((v >> 16) & e) == e ? 0u : v & 0xFFFF0000u);
}

// A place on the line of tiles: tile `tile` of the row tile `mt` of kv head `kvh` of sequence `seq` (-1: the prefix).
struct AttnAt {
    int seq, kvh, mt, tile, tiles, k0, keys;  // tile t holds the keys [k0 + 64 t, ...) below `keys`
};
__device__ __forceinline__ int own_tiles(const AttnArgs &P, int b) {
    return (own_keys(P, b) - own_cut(P, b) + kAtKeys - 1) / kAtKeys;
}
__device__ __forceinline__ void attn_step(const AttnArgs &P, AttnAt &a) {
    if (++a.tile < a.tiles) return;
    a.tile = 0;
    if (++a.mt < (a.seq < 0 ? P.mt_pre : P.mt_own)) return;
    a.mt = 0;
    if (++a.kvh < P.own.n_kv) return;
    a.kvh = 0;
    do {
        if (++a.seq >= P.own.n_seq) {  // behind the line: nothing reads this place
            a.seq = P.own.n_seq - 1;
            return;
        }
        a.keys = own_keys(P, a.seq);
        a.k0 = own_cut(P, a.seq);
        a.tiles = (a.keys - a.k0 + kAtKeys - 1) / kAtKeys;
    } while (a.tiles == 0);
}
// Number of the (problem, row tile) on the line.
__device__ __forceinline__ int attn_unit(const AttnArgs &P, const AttnAt &a) {
    return a.seq < 0 ? a.kvh * P.mt_pre + a.mt
                     : P.own.n_kv * P.mt_pre + (a.seq * P.own.n_kv + a.kvh) * P.mt_own + a.mt;
}
// Where CTA c's part begins.  No more CTAs share the line than it has tiles, so that no part is empty.
__device__ __forceinline__ long long line_part(long long total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int line_ctas(long long total, int ctas) { return (int)min((long long)ctas, max(total, 1ll)); }

// This CTA's part [first, end) of a line made of `line_pre` tiles of the prefix and, per sequence, tiles_of(b) * per_seq
// own ones; `seq` and `off` (tiles of the sequences before it): the sequence of the first tile, where it is an own one.
// CTA 0 writes the table of offsets.  False: no tile is this CTA's.  W: warps of the CTA, all of which call.
template <int W, typename F>
__device__ __forceinline__ bool line_share(int ns, F tiles_of, int per_seq, long long line_pre, int ctas, int *offs,
                                           long long &first, long long &end, int &seq, int &off) {
    __shared__ long long s_sum[W];
    __shared__ int s_seq, s_off;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x;
    long long units = 0;
    for (int b = tid; b < ns; b += W * 32) units += tiles_of(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    if (lane == 0) s_sum[warp] = units;
    __syncthreads();
    units = 0;
    for (int w = 0; w < W; ++w) units += s_sum[w];
    const long long total = line_pre + units * per_seq;
    const int nc = line_ctas(total, ctas);
    if (c >= nc) return false;
    first = line_part(total, nc, c);
    end = line_part(total, nc, c + 1);
    if (first >= line_pre || c == 0) {
        int run = 0;
        for (int b0 = 0; b0 < ns; b0 += W * 32) {
            const int b = b0 + tid, n = b < ns ? tiles_of(b) : 0;
            int x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) s_sum[warp] = x;
            __syncthreads();
            int at = run + x - n;
            for (int w = 0; w < W; ++w) {
                if (w < warp) at += (int)s_sum[w];
                run += (int)s_sum[w];
            }
            if (b < ns) {
                if (c == 0) offs[b] = at;
                const long long lo = line_pre + (long long)at * per_seq;
                if (n && first >= lo && first < lo + (long long)n * per_seq) {
                    s_seq = b;
                    s_off = at;
                }
            }
        }
        if (c == 0 && tid == 0) offs[ns] = run;
        __syncthreads();
        seq = s_seq;
        off = s_off;
    }
    return first < end;
}

template <int D>
constexpr int kAtStages = D == 64 ? 4 : D == 128 ? 3 : 2;
template <int D>
constexpr int kAtTileBytes = kAtKeys * D * 2;
template <int D>
constexpr int kAtMergeRow = D + 4;  // floats
template <int D>
constexpr int kAtSmem = 2 * kAtStages<D> * kAtTileBytes<D> + 32 * kAtMergeRow<D> * 4 + (D == 256 ? 64 * D * 2 : 0);

// Loads the tile at `a` into one stage, slots behind the last in use as zeros (V of a weight 0 must not be NaN).
template <int D>
__device__ __forceinline__ void attn_load(const AttnArgs &P, const AttnAt &a, uint32_t stage) {
    constexpr int C = D / 8, KPI = kAtThreads / C;  // 16-byte pieces of a key, keys per pass
    const KvArgs &kv = a.seq < 0 ? P.pre : P.own;
    const int c = threadIdx.x % C, k0 = threadIdx.x / C;
    const int t0 = a.k0 + a.tile * kAtKeys, left = a.keys - t0;
    const long long at = (a.seq < 0 ? 0 : (long long)a.seq * kv.seq_stride) + a.kvh * kv.head_stride + t0 * kv.slot_stride + c * 8;
    const uint16_t *k = kv.k + at, *v = kv.v + at;
#pragma unroll
    for (int j = 0; j < kAtKeys / KPI; ++j) {
        const int key = k0 + j * KPI;
        const bool in = key < left;
        const long long o = in ? key * kv.slot_stride : 0;
        const uint32_t dst = stage + key * (D * 2) + ((c ^ (key & 7)) << 4);
        cp16(dst, k + o, in ? 16 : 0);
        cp16(dst + kAtTileBytes<D>, v + o, in ? 16 : 0);
    }
}

template <int D>
struct AttnAcc {
    float o[D / 8][4], m[2], l[2];  // rows lane / 4 and lane / 4 + 8
};

// One warp's share of a tile: 16 rows x KPW keys from key `kw` of the tile on.
template <int D, bool BF16, bool F32, int KPW>
__device__ __forceinline__ void attn_tile(const AttnArgs &P, const AttnAt &a, AttnAcc<D> &A, const uint32_t (&qf)[D == 256 ? 1 : D / 16][4],
                                          uint32_t q_smem, uint32_t ks, uint32_t vs, const uint8_t *v_gen, int kw, int r0, int M) {
    const int lane = threadIdx.x & 31;
    float s[KPW / 8][4];
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
    const int krow = kw + ((lane >> 4) << 3) + (lane & 7), kc = (lane >> 3) & 1;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t af[4];
        if (D == 256) {
            const int row = lane & 15;
            ldm4(af, q_smem + row * (D * 2) + (((kk * 2 + (lane >> 4)) ^ (row & 7)) << 4));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) af[e] = qf[D == 256 ? 0 : kk][e];
        }
#pragma unroll
        for (int n = 0; n < KPW / 16; ++n) {
            uint32_t b[4];
            const int key = krow + n * 16;
            ldm4(b, ks + key * (D * 2) + (((kk * 2 + kc) ^ (key & 7)) << 4));
            mma16<BF16>(s[2 * n], af, b[0], b[1]);
            mma16<BF16>(s[2 * n + 1], af, b[2], b[3]);
        }
    }
    const int t0 = a.k0 + a.tile * kAtKeys + kw, col = (lane & 3) * 2;
    const bool prefix = a.seq < 0;
    const int base = prefix ? a.keys : P.base[a.seq];
    const bool open = t0 + KPW <= min(base, a.keys);  // every row sees every key of the range
    unsigned long long mask[2] = {0, 0};
    bool any_hidden = false;
    if (!open) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = r0 + (lane >> 2) + 8 * j, i = r / P.G;
            if (!prefix && r < M) mask[j] = row_mask(P, a.seq * P.rows + i, i);
        }
        any_hidden = !prefix && (P.rows > 1 || P.mask);
    }
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = s[n][e] * P.scale2;
            if (!open) {
                const int t = t0 + n * 8 + col + (e & 1);
                const bool seen = t < a.keys && (t < base || ((mask[e >> 1] >> (t - base)) & 1ull));
                x = seen ? x : -INFINITY;
            }
            s[n][e] = x;
        }
    if (P.scores && !prefix) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = r0 + (lane >> 2) + 8 * j;
            if (r < M) {
                float *to = P.scores + (((long long)a.seq * P.own.n_kv + a.kvh) * ((long long)P.rows * P.G) + r) * P.own.cap;
#pragma unroll
                for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = t0 + n * 8 + col + e;
                        if (t < a.keys) to[t] = s[n][2 * j + e];
                    }
            }
        }
    }
    // running maximum and sum
    float mb[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float mx = A.m[j];
#pragma unroll
        for (int n = 0; n < KPW / 8; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * j], s[n][2 * j + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float ms = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: weights 2^(-inf - 0) = 0
        const float f = ex2(A.m[j] - ms);
        A.m[j] = mx;
        A.l[j] *= f;
        mb[j] = ms - kAtLift<BF16>;
        if (f != 1.0f) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                A.o[d][2 * j] *= f;
                A.o[d][2 * j + 1] *= f;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[n][e] = ex2(s[n][e] - mb[e >> 1]);
            A.l[e >> 1] += s[n][e];
        }
    // Values that some row must not see can be infinite or NaN, and 0 x inf is not 0: in a range that holds such
    // values the products take zeros for them, and the rows that do see them add them one by one afterwards.
    bool odd = false;
    if (any_hidden) {
        for (int x = lane; x < KPW * (D / 2); x += 32) {
            const int key = kw + x / (D / 2), w = x % (D / 2);
            const uint32_t v = *reinterpret_cast<const uint32_t *>(v_gen + key * (D * 2) + (((w >> 2) ^ (key & 7)) << 4) + (w & 3) * 4);
            odd |= finite16<BF16>(v) != v;
        }
        odd = __any_sync(0xffffffffu, odd);
    }
    const int vrow = kw + (((lane >> 3) & 1) << 3) + (lane & 7), vc = lane >> 4;
#pragma unroll
    for (int kb = 0; kb < KPW / 16; ++kb) {
        constexpr int T = kAtTerms<BF16, F32>;
        uint32_t pf[T][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = s[2 * kb + (e >> 1)][2 * (e & 1)], y = s[2 * kb + (e >> 1)][2 * (e & 1) + 1];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                pf[t][e] = pack16<BF16>(x, y);
                x -= low16<BF16>(pf[t][e]);
                y -= high16<BF16>(pf[t][e]);
            }
        }
        const int key = vrow + kb * 16;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t b[4];
            ldm4t(b, vs + key * (D * 2) + (((d * 2 + vc) ^ (key & 7)) << 4));
            if (odd)
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = finite16<BF16>(b[e]);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                mma16<BF16>(A.o[2 * d], pf[t], b[0], b[1]);
                mma16<BF16>(A.o[2 * d + 1], pf[t], b[2], b[3]);
            }
        }
    }
    if (!odd) return;
    for (int key = 0; key < KPW; ++key) {
        float p[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < KPW / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n * 8 + (e & 1) == (key & ~7) + (key & 1)) p[e >> 1] = s[n][e];
        const int t = t0 + key, from = (lane & ~3) | ((key & 7) >> 1);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            p[j] = __shfl_sync(0xffffffffu, p[j], from);
            if (t >= a.keys || (t >= base && !((mask[j] >> (t - base)) & 1ull))) continue;
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {
                const uint32_t v = *reinterpret_cast<const uint32_t *>(v_gen + (kw + key) * (D * 2) + ((d ^ ((kw + key) & 7)) << 4) +
                                                                       (lane & 3) * 4);
                const uint32_t bad = v ^ finite16<BF16>(v);
                if (bad & 0xFFFFu) A.o[d][2 * j] = fmaf(p[j], low16<BF16>(v), A.o[d][2 * j]);
                if (bad >> 16) A.o[d][2 * j + 1] = fmaf(p[j], high16<BF16>(v), A.o[d][2 * j + 1]);
            }
        }
    }
}

template <int D, bool BF16, bool F32>
__global__ void __launch_bounds__(kAtThreads) attn_split_kernel(const AttnArgs P) {
    extern __shared__ __align__(128) uint8_t at_smem[];
    constexpr int NS = kAtStages<D>, TB = kAtTileBytes<D>, MR = kAtMergeRow<D>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x;
    griddep_launch_dependents();
    const int nkv = P.own.n_kv, per_seq = nkv * P.mt_own;
    const int tp = P.mt_pre ? (P.prefix_len - P.cut_pre + kAtKeys - 1) / kAtKeys : 0;
    const long long line_pre = (long long)nkv * P.mt_pre * tp;
    long long first, end;
    int seq = 0, off = 0;
    if (!line_share<kAtThreads / 32>(P.own.n_seq, [&](int b) { return own_tiles(P, b); }, per_seq, line_pre, P.ctas, P.offs, first, end,
                                     seq, off)) {
        griddep_wait();
        return;
    }
    AttnAt at;
    if (first < line_pre) {
        at.seq = -1;
        at.keys = P.prefix_len;
        at.k0 = P.cut_pre;
        at.tiles = tp;
        const int u = (int)(first / tp);
        at.kvh = u / P.mt_pre;
        at.mt = u % P.mt_pre;
        at.tile = (int)(first % tp);
    } else {
        at.seq = seq;
        at.keys = own_keys(P, seq);
        at.k0 = own_cut(P, seq);
        at.tiles = own_tiles(P, seq);
        const long long in = first - line_pre - (long long)off * per_seq;
        const int u = (int)(in / at.tiles);
        at.kvh = u / P.mt_own;
        at.mt = u % P.mt_own;
        at.tile = (int)(in % at.tiles);
    }
    const uint32_t smem = smem_u32(at_smem);
    float *merge = reinterpret_cast<float *>(at_smem + 2 * NS * TB);
    float2(*s_ml)[16] = reinterpret_cast<float2(*)[16]>(merge);  // the warps' statistics, before their outputs
    const uint32_t q_smem = smem + 2 * NS * TB + 32 * MR * 4;
    AttnAt ahead = at;
    const int steps = (int)(end - first);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        if (s < steps) {
            attn_load<D>(P, ahead, smem + s * 2 * TB);
            attn_step(P, ahead);
        }
        cp_commit();
    }
    AttnAcc<D> A;
    uint32_t qf[D == 256 ? 1 : D / 16][4];
    bool fresh = true;
    int stage = 0, M = 0, r0 = 0, wm = 1, wi = 0, wk = 0;
    for (int s = 0; s < steps; ++s) {
        if (fresh) {  // a new (problem, row tile): its query vectors, empty statistics
            fresh = false;
            const int rt = at.seq < 0 ? P.rt_pre : P.rt_own, row0 = at.seq < 0 ? 0 : at.seq * P.rows;
            M = (at.seq < 0 ? P.S : P.rows) * P.G;
            wm = rt >> 4;
            wi = warp % wm;
            wk = warp / wm;
            r0 = at.mt * rt + wi * 16;
            if (D == 256) {
                __syncthreads();
                for (int x = tid; x < rt * (D / 8); x += kAtThreads) {
                    const int row = x / (D / 8), ch = x % (D / 8), r = at.mt * rt + row;
                    uint4 val = make_uint4(0, 0, 0, 0);
                    if (r < M)
                        val = *reinterpret_cast<const uint4 *>(P.q + ((long long)(row0 + r / P.G) * P.H + at.kvh * P.G + r % P.G) * D + ch * 8);
                    *reinterpret_cast<uint4 *>(at_smem + (q_smem - smem) + row * (D * 2) + ((ch ^ (row & 7)) << 4)) = val;
                }
                // the tile's barrier below orders these writes before their readers
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = r0 + (lane >> 2) + 8 * j;
                    const uint16_t *src = P.q + ((long long)(row0 + r / P.G) * P.H + at.kvh * P.G + r % P.G) * D + (lane & 3) * 2;
#pragma unroll
                    for (int kk = 0; kk < (D == 256 ? 1 : D / 16); ++kk)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            qf[kk][j + 2 * e] = r < M ? *reinterpret_cast<const uint32_t *>(src + kk * 16 + e * 8) : 0u;
                }
            }
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) A.o[d][e] = 0.0f;
            A.m[0] = A.m[1] = -INFINITY;
            A.l[0] = A.l[1] = 0.0f;
        }
        cp_wait<NS - 2>();
        __syncthreads();
        {
            const int next = stage == 0 ? NS - 1 : stage - 1;  // the stage of the tile before this one is free now
            if (s + NS - 1 < steps) {
                attn_load<D>(P, ahead, smem + next * 2 * TB);
                attn_step(P, ahead);
            }
            cp_commit();
        }
        const uint32_t ks = smem + stage * 2 * TB, vs = ks + TB, qs = q_smem + wi * 16 * D * 2;
        const uint8_t *vg = at_smem + stage * 2 * TB + TB;
        if (r0 < M) {
            if (wm == 1)
                attn_tile<D, BF16, F32, 16>(P, at, A, qf, qs, ks, vs, vg, wk * 16, r0, M);
            else if (wm == 2)
                attn_tile<D, BF16, F32, 32>(P, at, A, qf, qs, ks, vs, vg, wk * 32, r0, M);
            else if (D < 256) {
                attn_tile<D, BF16, F32, D < 256 ? 64 : 32>(P, at, A, qf, qs, ks, vs, vg, 0, r0, M);
            } else {  // half of the tile at a time: 128 registers of a thread hold the output
                attn_tile<D, BF16, F32, 32>(P, at, A, qf, qs, ks, vs, vg, 0, r0, M);
                attn_tile<D, BF16, F32, 32>(P, at, A, qf, qs, ks, vs, vg, 32, r0, M);
            }
        }
        stage = stage + 1 == NS ? 0 : stage + 1;
        const bool last = s + 1 == steps || at.tile + 1 == at.tiles;
        if (last) {  // one partial result of this (problem, row tile)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                A.l[j] += __shfl_xor_sync(0xffffffffu, A.l[j], 1);
                A.l[j] += __shfl_xor_sync(0xffffffffu, A.l[j], 2);
            }
            const long long slot = (long long)attn_unit(P, at) + c;
            float *part = P.part + slot * P.rt_max * D;
            float2 *ml = P.ml + slot * P.rt_max;
            if (wm == 4) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = wi * 16 + (lane >> 2) + 8 * j;
                    if (r0 + (lane >> 2) + 8 * j < M) {
                        if ((lane & 3) == 0) ml[row] = make_float2(A.m[j], A.l[j]);
#pragma unroll
                        for (int d = 0; d < D / 8; ++d)
                            *reinterpret_cast<float2 *>(part + (long long)row * D + d * 8 + (lane & 3) * 2) = make_float2(A.o[d][2 * j], A.o[d][2 * j + 1]);
                    }
                }
            } else {  // the warps that share rows add theirs up in a fixed order
                if ((lane & 3) == 0) {
                    s_ml[warp][lane >> 2] = make_float2(A.m[0], A.l[0]);
                    s_ml[warp][(lane >> 2) + 8] = make_float2(A.m[1], A.l[1]);
                }
                __syncthreads();
                const int wn = 4 / wm;
                float f[2], mm[2], ll[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = (lane >> 2) + 8 * j;
                    float m = -INFINITY, l = 0.0f;
                    for (int w = 0; w < wn; ++w) m = fmaxf(m, s_ml[w * wm + wi][row].x);
                    const float ms = m == -INFINITY ? 0.0f : m;
                    for (int w = 0; w < wn; ++w) l += s_ml[w * wm + wi][row].y * ex2(s_ml[w * wm + wi][row].x - ms);
                    f[j] = ex2(A.m[j] - ms);
                    mm[j] = m;
                    ll[j] = l;
                }
                __syncthreads();
                for (int w = 0; w < wn; ++w) {
                    if (wk == w) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float2 *to = reinterpret_cast<float2 *>(merge + (wi * 16 + (lane >> 2) + 8 * j) * MR + (lane & 3) * 2);
#pragma unroll
                            for (int d = 0; d < D / 8; ++d) {
                                float2 v = make_float2(A.o[d][2 * j] * f[j], A.o[d][2 * j + 1] * f[j]);
                                if (w) {
                                    const float2 u = to[d * 4];
                                    v.x += u.x;
                                    v.y += u.y;
                                }
                                to[d * 4] = v;
                            }
                        }
                    }
                    __syncthreads();
                }
                if (wk == 0 && (lane & 3) == 0)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (r0 + (lane >> 2) + 8 * j < M) ml[wi * 16 + (lane >> 2) + 8 * j] = make_float2(mm[j], ll[j]);
                const int have = min(wm * 16, M - at.mt * wm * 16);
                for (int x = tid; x < have * (D / 4); x += kAtThreads) {
                    const int row = x / (D / 4), ch = x % (D / 4);
                    *reinterpret_cast<float4 *>(part + (long long)row * D + ch * 4) = *reinterpret_cast<const float4 *>(merge + row * MR + ch * 4);
                }
            }
            fresh = true;
        }
        attn_step(P, at);
    }
    griddep_wait();  // the joining launch waits for this one alone, and needs the tensor-memory kernel's results too
}

// Partials of one (problem, row tile): those of the CTAs whose parts meet its stretch [u0, u1) of the line.
struct AttnParts {
    int unit, c0, n;  // partial j is at unit + c0 + j
};
__device__ __forceinline__ AttnParts attn_parts(int unit, long long u0, long long u1, long long total, int ctas) {
    AttnParts r{unit, 0, 0};
    if (u0 >= u1) return r;
    int a = (int)(u0 * ctas / total);
    while (a > 0 && line_part(total, ctas, a) > u0) --a;
    while (line_part(total, ctas, a + 1) <= u0) ++a;
    int b = (int)((u1 - 1) * ctas / total);
    while (b > 0 && line_part(total, ctas, b) > u1 - 1) --b;
    while (line_part(total, ctas, b + 1) <= u1 - 1) ++b;
    r.c0 = a;
    r.n = b - a + 1;
    return r;
}
// The lists of partials of row vector r (within its sequence) of a (sequence, kv head): of the prefix and its own slots,
// from this kernel (0, 1) and from the tensor-memory kernel (2, 3).
struct AttnRowParts {
    AttnParts list[4];
    int row[4], n;
};
__device__ __forceinline__ AttnRowParts attn_row_parts(const AttnArgs &P, int seq, int kvh, int r) {
    AttnRowParts R;
    const int nkv = P.own.n_kv, rp = seq * P.rows * P.G + r;
    {
        const int per_seq = nkv * P.mt_own, tp = P.mt_pre ? (P.prefix_len - P.cut_pre + kAtKeys - 1) / kAtKeys : 0;
        const long long line_pre = (long long)nkv * P.mt_pre * tp, total = line_pre + (long long)P.offs[P.own.n_seq] * per_seq;
        const int nc = line_ctas(total, P.ctas);
        const int up = kvh * P.mt_pre + rp / P.rt_pre;
        R.row[0] = rp % P.rt_pre;
        R.list[0] = attn_parts(up, (long long)up * tp, P.mt_pre ? (long long)(up + 1) * tp : 0, total, nc);
        const int off = P.offs[seq], tiles = P.offs[seq + 1] - off, uo = kvh * P.mt_own + r / P.rt_own;
        const long long lo = line_pre + (long long)off * per_seq + (long long)uo * tiles;
        R.row[1] = r % P.rt_own;
        R.list[1] = attn_parts(nkv * P.mt_pre + seq * per_seq + uo, lo, lo + tiles, total, nc);
    }
    R.list[2] = R.list[3] = AttnParts{0, 0, 0};
    R.row[2] = R.row[3] = 0;
    if (P.tc_pre || P.tc_own) {
        const int per_seq = nkv * P.tcm_own, tp = P.tc_pre ? P.cut_pre / P.tc_keys : 0;
        const long long line_pre = (long long)nkv * P.tcm_pre * tp, total = line_pre + (long long)P.tc_offs[P.own.n_seq] * per_seq;
        const int nc = line_ctas(total, P.tc_ctas);
        if (P.tc_pre) {
            const int rt = P.tc2_pre ? 128 : P.tc_rows, up = kvh * P.tcm_pre + rp / rt;
            R.row[2] = rp % rt;
            R.list[2] = attn_parts(up, (long long)up * tp, (long long)(up + 1) * tp, total, nc);
            R.list[2].n <<= P.tc2_pre;
        }
        if (P.tc_own) {
            const int rt = P.tc2_own ? 128 : P.tc_rows, uo = kvh * P.tcm_own + r / rt;
            const int off = P.tc_offs[seq], tiles = P.tc_offs[seq + 1] - off;
            const long long lo = line_pre + (long long)off * per_seq + (long long)uo * tiles;
            R.row[3] = r % rt;
            R.list[3] = attn_parts(nkv * P.tcm_pre + seq * per_seq + uo, lo, lo + tiles, total, nc);
            R.list[3].n <<= P.tc2_own;
        }
    }
    R.n = R.list[0].n + R.list[1].n + R.list[2].n + R.list[3].n;
    return R;
}
// Partial j of the row vector: its statistics and, in units of D floats, its output.
__device__ __forceinline__ const float2 *attn_part(const AttnArgs &P, const AttnRowParts &R, int j, const float *&out, int D) {
    const int n0 = R.list[0].n, n1 = n0 + R.list[1].n, n2 = n1 + R.list[2].n;
    if (j < n1) {
        const bool o = j >= n0;
        const long long at = (long long)(o ? R.list[1].unit + R.list[1].c0 + j - n0 : R.list[0].unit + R.list[0].c0 + j) * P.rt_max +
                             (o ? R.row[1] : R.row[0]);
        out = P.part + at * D;
        return P.ml + at;
    }
    const bool o = j >= n2;
    const int i = o ? j - n2 : j - n1, two = o ? P.tc2_own : P.tc2_pre;  // two halves of a partial follow one another
    const long long at = (long long)((o ? R.list[3].unit + R.list[3].c0 : R.list[2].unit + R.list[2].c0) + (i >> two)) * P.tc_rows +
                         (o ? R.row[3] : R.row[2]) + (two && (i & 1) ? 128 : 0);
    out = P.tc_part + at * D;
    return P.tc_ml + at;
}

// Joins the partials: CTAs [0, S x H) one row vector each; with acc, further CTAs 256 slots of one (sequence, kv head) each.
template <int D, bool BF16>
__global__ void __launch_bounds__(kAtCombine) attn_join_kernel(const AttnArgs P, int chunks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    __shared__ float s_m[4], s_l[4];
    if (blockIdx.x < (unsigned)(P.S * P.H)) {
        constexpr int E = D / 32;
        __shared__ float s_o[4][D];
        const int row = blockIdx.x / P.H, h = blockIdx.x % P.H, seq = row / P.rows, kvh = h / P.G;
        if (P.base[seq] < 0) return;
        const AttnRowParts R = attn_row_parts(P, seq, kvh, (row % P.rows) * P.G + h % P.G);
        const int n = R.n;
        const float *src;
        float m = -INFINITY;
        for (int j = threadIdx.x; j < n; j += kAtCombine) m = fmaxf(m, attn_part(P, R, j, src, D)->x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) s_m[warp] = m;
        __syncthreads();
        m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        if (m == -INFINITY) m = 0.0f;
        float o[E] = {}, l = 0.0f;
#pragma unroll 4
        for (int j = warp; j < n; j += 4) {
            const float2 ml = *attn_part(P, R, j, src, D);
            const float f = ex2(ml.x - m);
            l = fmaf(ml.y, f, l);
            src += lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 v = *reinterpret_cast<const float2 *>(src + e);
                o[e] = fmaf(v.x, f, o[e]);
                o[e + 1] = fmaf(v.y, f, o[e + 1]);
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
        if (lane == 0) s_l[warp] = l;
        __syncthreads();
        l = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const long long to = (long long)blockIdx.x * D;
        for (int d = threadIdx.x * 2; d < D; d += kAtCombine * 2) {
            const float x = ((s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d])) * inv;
            const float y = ((s_o[0][d + 1] + s_o[1][d + 1]) + (s_o[2][d + 1] + s_o[3][d + 1])) * inv;
            if (P.out_f32)
                *reinterpret_cast<float2 *>(static_cast<float *>(P.out) + to + d) = make_float2(x, y);
            else
                *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(P.out) + to + d) = pack16<BF16>(x, y);
        }
        return;
    }
    // acc[slot] += sum over the group's row vectors of 2^(x - m) / l
    const int u = blockIdx.x - P.S * P.H, g = u / chunks, chunk = u % chunks;
    const int seq = g / P.own.n_kv, kvh = g % P.own.n_kv;
    const int keys = own_keys(P, seq);
    const int t0 = chunk * 2 * kAtCombine;
    if (t0 >= keys) return;
    __shared__ float2 s_row[64];  // m and 1 / l of the row vectors
    const int M = P.rows * P.G;
    float sum[2] = {0.0f, 0.0f};
    for (int r0 = 0; r0 < M; r0 += 64) {
        __syncthreads();
        for (int r = r0 + warp; r < min(M, r0 + 64); r += 4) {
            const AttnRowParts R = attn_row_parts(P, seq, kvh, r);
            const int n = R.n;
            const float *src;
            float m = -INFINITY, l = 0.0f;
            for (int j = lane; j < n; j += 32) m = fmaxf(m, attn_part(P, R, j, src, D)->x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (m == -INFINITY) m = 0.0f;
            for (int j = lane; j < n; j += 32) {
                const float2 ml = *attn_part(P, R, j, src, D);
                l = fmaf(ml.y, ex2(ml.x - m), l);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane == 0) s_row[r - r0] = make_float2(m - kAtLift<BF16>, l == 0.0f ? 0.0f : 1.0f / l);
        }
        __syncthreads();
        const float *x = P.scores + ((long long)g * M + r0) * P.own.cap + t0 + threadIdx.x;
        for (int r = 0; r < min(M - r0, 64); ++r, x += P.own.cap) {
            const float2 st = s_row[r];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (t0 + j * kAtCombine + (int)threadIdx.x < keys) {
                    const float w = x[j * kAtCombine];
                    if (w != -INFINITY) sum[j] = fmaf(ex2(w - st.x), st.y, sum[j]);
                }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = t0 + j * kAtCombine + threadIdx.x;
        if (t < keys) P.own.acc[(long long)g * P.own.cap + t] += sum[j];
    }
}

}  // namespace pgb
