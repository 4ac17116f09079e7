// Attention of a batch behind a shared prefix: out = softmax(scale q.k) v.
//
// Problems: the prefix, once per kv head, with the rows of ALL sequences (its keys are read once for the batch), and every
// sequence's own slots per kv head with that sequence's rows.  A problem has M = rows x group query vectors.  Where M is
// large it goes to the tensor-memory kernel (kernels_attn_tc.cuh); this kernel takes the others in row tiles of 8 or 16.  Work is counted in tiles of 64 keys; all tiles of all problems form one line, and CTA c of
// n takes the c-th equal part of it, whatever the lengths (read on the device): no sequence is too long or too short.  Within its part
// a CTA keeps the running maximum m, sum l and output of one problem at a time (log2 units)
//     m' = max(m, x),  l' = l 2^(m-m') + sum 2^(x-m'),  o' = o 2^(m-m') + sum 2^(x-m') v,   x = scale log2(e) q.k
// and writes them as one partial result when the problem or the part ends.  A last launch joins the partials of a row in
// the order of the CTAs (no atomics) and adds up the weights that the slots received.
//
// Few rows per key make this bound by HBM: four warps share a tile, 16 keys each, while a fifth keeps the copy engine
// filling the other stages.  With up to 8 query vectors (a group of one decode row) only half of a matrix instruction's 16
// rows would be used, so the second product is turned round: O^T = V^T P^T has the query vectors in its 8 columns, which
// the scores' registers already fit, and halves its instructions and registers.  Measured: 2 x 32 heads over up to 50000 slots
// (8 key heads of 128, fp32 out with weights kept) 57 us, 5.4 TB/s of the 6.5 that a copy reaches; 32 x 64 heads over up to 2048
// slots 37 us, 4.3 TB/s (a CTA's parts are 11 tiles there, and each change of the problem exposes its loads).
#pragma once
#include "kernels_norm_rope.cuh"

namespace pgb {

constexpr int kAtKeys = 64;      // keys of a tile
constexpr int kAtThreads = 160;  // 4 warps with 16 keys of a tile each, one that issues the copies
constexpr int kAtCombine = 128;
constexpr int kTcKeys = 64;  // keys of a tile of the tensor-memory kernel
// Row vectors of a problem up to which attn_split_kernel takes it, and the joining launch adds up the weights itself.  us of a
// call with 4 key heads, bf16, fp32 out, by that kernel / by the one on tensor memory:
//                              12 row vectors     20 row vectors
//   D = 64,  1 x 20000 slots    17.5 / 24.3        19.1 / 24.3
//   D = 64,  8 x 4000           15.4 / 19.9        18.7 / 20.2
//   D = 128, 1 x 20000          24.7 / 27.1        27.6 / 27.6
//   D = 128, 8 x 4000           24.9 / 22.9        29.8 / 23.2
//   D = 256, 1 x 20000          43.9 / 28.7        71.3 / 28.8
//   D = 256, 8 x 4000           51.5 / 27.3        71.9 / 29.4
// and of 12 and 20 rows behind 2000 keys (D = 128): 11.5 / 15.6, 14.7 / 16.2.  The border suits D = 128; at D = 256, where a row tile of
// 16 takes all 255 registers and spills 500 bytes, up to 8 (26.1 us for 8 x 4000) the split kernel keeps up, beyond not.
constexpr int kAtMany = 16;
constexpr int kAtChunk = 1024;  // slots whose weights one CTA adds up

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
    int mt_pre, mt_own;          // row tiles of a problem (mt_pre 0: no prefix)
    // the tensor-memory kernel
    int tc_pre, tc_own;    // whether it takes the prefix, the own slots
    int tc_ctas, tc_rows;  // its CTAs, rows of one of its partials
    int tcm_pre, tcm_own;  // its row tiles of a problem
    int tc2_pre, tc2_own;  // 1: a row tile has 128 rows and its keys go to two halves of a partial in turn
    int *err;
    // scratch.  A (problem, row tile) is a unit; partial `unit + c` is that of CTA c, and no two pairs share a sum, since
    // both only grow along the line.
    float *part;    // [units + ctas][row tile][D], then [units + tc_ctas][tc_rows][D]: outputs, unnormalised
    float2 *ml;     // one per row of part: m and l
    long long tc_row0;      // first row of the tensor-memory kernel's
    int2 *cta_of, *tc_cta_of;  // per unit: the CTAs that have its first and its last tile
    // x of the own slots (-inf: not seen), only with acc: [n_seq][n_kv][rows * G][cap] from the split kernel,
    // [n_seq][n_kv][cap / 4, rounded up][rows * G][4] from the tensor-memory kernel, whose lanes hold neighbouring rows
    float *scores;
    float2 *stats;  // [S * H]: m and 1 / l of every row vector, joined; only with acc and many rows
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
// Where the tensor-memory kernel's scores of slot 4 q and the three behind it with row vector r stand.
__device__ __forceinline__ float *score_at(const AttnArgs &P, int g, int q, int M, int r) {
    return P.scores + (((long long)g * ((P.own.cap + 3) >> 2) + q) * M + r) * 4;
}
// New slots that row i of a sequence sees, a bit each.
__device__ __forceinline__ unsigned long long row_mask(const AttnArgs &P, int row, int i) {
    const unsigned long long in = P.rows == 64 ? ~0ull : (1ull << P.rows) - 1;
    return (P.mask ? P.mask[row] : ~0ull >> (63 - i)) & in;
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
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Weights enter the second product in 16-bit terms.  A 16-bit output needs one (its own rounding is as large).  An fp32
// output takes two of f16 or three of bf16.  Rounded to nearest these leave 2^-22 or 2^-24 of a weight, cut off (as the
// tensor-memory kernel does) 2^-21 or 2^-22.  f16 weights are scaled by 2^6 against underflow of their lower term: its steps of
// 2^-24 leave up to 2^-31 of the largest weight, or 2^-30 where a first term below 2^-14 was rounded too.  With the 2^8 that
// the maximum may lag behind, weights stay below 2^15; l carries the same factor, so it cancels.  More of one is less of the other: with 2^10 and
// 2^5 (2^-34 of the largest) an f16 batch of 32 x 64 heads behind 32768 keys took 100.1 us, with 2^13 and 2^2 106.3, with these 96.2.
template <bool BF16>
constexpr float kAtLift = BF16 ? 0.0f : 6.0f;
constexpr float kAtLag = 8.0f;  // log2 by which a row's maximum may grow before o, l and m are rescaled
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
    int seq, kvh, mt, tile, tiles, keys, base;  // tile t holds the keys [64 t, ...) below `keys`
};
__device__ __forceinline__ int own_tiles(const AttnArgs &P, int b) { return P.tc_own ? 0 : (own_keys(P, b) + kAtKeys - 1) / kAtKeys; }
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
        a.base = P.base[a.seq];
        a.keys = own_keys(P, a.seq);
        a.tiles = own_tiles(P, a.seq);
    } while (a.tiles == 0);
}
// Number of the (problem, row tile) on the line.
__device__ __forceinline__ int attn_unit(const AttnArgs &P, const AttnAt &a) {
    return a.seq < 0 ? a.kvh * P.mt_pre + a.mt
                     : P.own.n_kv * P.mt_pre + (a.seq * P.own.n_kv + a.kvh) * P.mt_own + a.mt;
}
// Where CTA c's part begins.  No more CTAs share the line than leave each `least` tiles: none is empty, and the shorter the
// parts, the more partial results there are to join.
__device__ __forceinline__ long long line_part(long long total, int ctas, int c) { return total * c / ctas; }
__device__ __forceinline__ int line_ctas(long long total, int ctas, int least) { return (int)min((long long)ctas, max(total / least, 1ll)); }

// This CTA's part [first, end) of a line made of `line_pre` tiles of the prefix and, per sequence, tiles_of(b) * per_seq
// own ones; `seq` and `off` (tiles of the sequences before it): the sequence of the first tile, where it is an own one.
// False: no tile is this CTA's.  W: warps of the CTA, all of which call.
template <int W, typename F>
__device__ __forceinline__ bool line_share(int ns, F tiles_of, int per_seq, long long line_pre, int ctas, int least, long long &first,
                                           long long &end, int &seq, int &off) {
    __shared__ int s_sum[W], s_seq, s_off;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x;
    const int mine0 = tid < ns ? tiles_of(tid) : 0;
    long long units = 0;
    if (ns <= 32) {  // every warp for itself
        units = __reduce_add_sync(0xffffffffu, lane == tid || lane >= ns ? (lane < ns ? mine0 : 0) : tiles_of(lane));
    } else {
        int sum = mine0;
        for (int b = tid + W * 32; b < ns; b += W * 32) sum += tiles_of(b);
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        for (int w = 0; w < W; ++w) units += s_sum[w];
    }
    const long long total = line_pre + units * per_seq;
    const int nc = line_ctas(total, ctas, least);
    if (c >= nc) return false;
    first = line_part(total, nc, c);
    end = line_part(total, nc, c + 1);
    if (first >= line_pre && first < end) {
        int run = 0;
        for (int b0 = 0; b0 < ns; b0 += W * 32) {
            const int b = b0 + tid, n = b0 == 0 ? mine0 : b < ns ? tiles_of(b) : 0;
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
                if (w < warp) at += s_sum[w];
                run += s_sum[w];
            }
            const long long lo = line_pre + (long long)at * per_seq;
            if (n && first >= lo && first < lo + (long long)n * per_seq) {
                s_seq = b;
                s_off = at;
            }
        }
        __syncthreads();
        seq = s_seq;
        off = s_off;
    }
    return first < end;
}

template <int D, int RT>
struct SplitShape {
    static constexpr int PER_SM = D == 64 ? 3 : D == 128 ? (RT == 8 ? 3 : 2) : 1;
    static constexpr int STAGES = D == 64 ? 4 : D == 128 ? (RT == 8 ? 2 : 3) : 3;
    static constexpr int TILE = kAtKeys * D * 2;  // bytes of a tile of keys or values: [D / 64][64 keys][128 swizzled bytes]
    static constexpr int MERGE_ROW = D + 4;       // floats
    static constexpr int SMEM = 1024 + 2 * STAGES * TILE + RT * MERGE_ROW * 4;
};

// Registers of one warp's row tile.  Row tile 16: o[d][..] has 8 dims x rows lane / 4, + 8; m and l of the same rows.
// Row tile 8: o[d][..] has 16 dims (lane / 4, + 8) x rows 2 (lane % 4), + 1; m and l of row lane / 4.
template <int D, int RT>
struct AttnAcc {
    float o[RT == 16 ? D / 8 : D / 16][4], m[RT / 8], l[RT / 8];
};

__device__ __forceinline__ uint32_t tile_at(int key, int chunk) {  // byte of a 16-byte piece of a key
    return (uint32_t)((chunk >> 3) * (kAtKeys * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
}

// One warp's share of a tile: its 16 keys from key `kw` on.
template <int D, bool BF16, bool F32, int RT>
__device__ __forceinline__ void attn_tile(const AttnArgs &P, const AttnAt &a, AttnAcc<D, RT> &A, const uint32_t (&qf)[D / 16][RT / 4],
                                          uint32_t ks, uint32_t vs, int kw, int r0, int M) {
    constexpr int T = kAtTerms<BF16, F32>, J = RT / 8;
    const int lane = threadIdx.x & 31;
    float s[2][4] = {};
    {
        const int key = kw + ((lane >> 4) << 3) + (lane & 7), kc = (lane >> 3) & 1;
        float s2[2][4] = {};  // two chains each: the sums of even and odd steps
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t b[4], af[4] = {qf[kk][0], 0u, qf[kk][RT == 16 ? 2 : 1], 0u};
            if (RT == 16) {
                af[1] = qf[kk][1 % (RT / 4)];
                af[3] = qf[kk][3 % (RT / 4)];
            }
            ldm4(b, ks + tile_at(key, kk * 2 + kc));
            mma16<BF16>(kk & 1 ? s2[0] : s[0], af, b[0], b[1]);
            mma16<BF16>(kk & 1 ? s2[1] : s[1], af, b[2], b[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2 * J; ++e) s[n][e] = (s[n][e] + s2[n][e]) * P.scale2;
    }
    const int t0 = a.tile * kAtKeys + kw, col = (lane & 3) * 2;
    const bool open = t0 + 16 <= min(a.base, a.keys);  // every row sees every key of the range
    uint32_t seen = 0;  // bit 4 n + e: whether s[n][e]'s row sees its key
    if (!open) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int r = r0 + (lane >> 2) + 8 * j, i = r / P.G;
            const unsigned long long mask = a.seq >= 0 && r < M ? row_mask(P, a.seq * P.rows + i, i) : 0;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int t = t0 + n * 8 + col + e;
                    if (t < a.keys && (t < a.base || ((mask >> (t - a.base)) & 1ull)))
                        seen |= 1u << (4 * n + 2 * j + e);
                    else
                        s[n][2 * j + e] = -INFINITY;
                }
        }
    }
    if (P.scores && a.seq >= 0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int r = r0 + (lane >> 2) + 8 * j;
            if (r < M) {
                float *to = P.scores + (((long long)a.seq * P.own.n_kv + a.kvh) * ((long long)P.rows * P.G) + r) * P.own.cap;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int t = t0 + n * 8 + col + e;
                        if (t < a.keys) to[t] = s[n][2 * j + e];
                    }
            }
        }
    }
    // The maximum only has to keep the weights in range, and cancels in o / l.
    float f[J];
    bool moved = false;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        float top = fmaxf(fmaxf(s[0][2 * j], s[0][2 * j + 1]), fmaxf(s[1][2 * j], s[1][2 * j + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        f[j] = 1.0f;
        if (top > A.m[j] + kAtLag) {
            f[j] = ex2(A.m[j] - top);
            A.m[j] = top;
            A.l[j] *= f[j];
            moved = true;
        }
    }
    if (__any_sync(0xffffffffu, moved)) {
        if (RT == 16) {
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) A.o[RT == 16 ? d : 0][e] *= f[(e >> 1) % J];
        } else {
            const float f0 = __shfl_sync(0xffffffffu, f[0], (lane & 3) * 8), f1 = __shfl_sync(0xffffffffu, f[0], (lane & 3) * 8 + 4);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) A.o[d][e] *= e & 1 ? f1 : f0;
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float ms = (A.m[j] == -INFINITY ? 0.0f : A.m[j]) - kAtLift<BF16>;  // nothing seen yet: weights 2^(-inf - 0) = 0
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[n][2 * j + e] = ex2(s[n][2 * j + e] - ms);
                A.l[j] += s[n][2 * j + e];
            }
    }
    // Values that some row does not see (or that were never stored) can be infinite or NaN, and 0 x inf is not 0: in a range
    // that holds such values the products take zeros for them, and the rows that do see them add them one by one afterwards.
    bool odd = false;
    if (!open) {
        const int key = kw + (lane & 15);
        for (int ch = lane >> 4; ch < D / 8; ch += 2) {
            uint32_t v[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(vs + tile_at(key, ch)));
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= finite16<BF16>(v[e]) != v[e];
        }
        odd = __any_sync(0xffffffffu, odd);
    }
    // the weights in T terms: pf[t][0, 1] of keys 0-7 and [2, 3] of keys 8-15, rows lane / 4 and + 8
    uint32_t pf[T][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < J; ++j) {
            float x = s[n][2 * j], y = s[n][2 * j + 1];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                pf[t][2 * n + j] = pack16<BF16>(x, y);
                x -= low16<BF16>(pf[t][2 * n + j]);
                y -= high16<BF16>(pf[t][2 * n + j]);
            }
        }
    if (RT == 16) {
        const int key = kw + (((lane >> 3) & 1) << 3) + (lane & 7), vc = lane >> 4;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t b[4];
            ldm4t(b, vs + tile_at(key, d * 2 + vc));
            if (odd)
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = finite16<BF16>(b[e]);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                mma16<BF16>(A.o[RT == 16 ? 2 * d : 0], pf[t], b[0], b[1]);
                mma16<BF16>(A.o[RT == 16 ? 2 * d + 1 : 0], pf[t], b[2], b[3]);
            }
        }
    } else {
        const int key = kw + ((lane >> 4) << 3) + (lane & 7), vc = (lane >> 3) & 1;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t v[4];
            ldm4t(v, vs + tile_at(key, d * 2 + vc));
            if (odd)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = finite16<BF16>(v[e]);
#pragma unroll
            for (int t = 0; t < T; ++t) mma16<BF16>(A.o[d], v, pf[t][0], pf[t][2]);
        }
    }
    if (!odd) return;
    for (int key = 0; key < 16; ++key) {
        const int n = key >> 3, e = key & 1, from = (lane & ~3) | ((key & 7) >> 1);  // the lane of this row with the key's weight
        float p[2];
        bool see[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float w = j < J ? (n ? (e ? s[1][(2 * j + 1) & 3] : s[1][(2 * j) & 3]) : (e ? s[0][(2 * j + 1) & 3] : s[0][(2 * j) & 3])) : 0.0f;
            p[j] = __shfl_sync(0xffffffffu, w, from);
            see[j] = (__shfl_sync(0xffffffffu, seen, from) >> (4 * n + 2 * j + e)) & 1u;
        }
        if (RT == 8) {  // o has the rows 2 (lane % 4), + 1
            const float w = p[0];
            const int sw = see[0];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                p[j] = __shfl_sync(0xffffffffu, w, (2 * (lane & 3) + j) * 4);
                see[j] = __shfl_sync(0xffffffffu, sw, (2 * (lane & 3) + j) * 4);
            }
        }
#pragma unroll
        for (int d = 0; d < (RT == 16 ? D / 8 : D / 16); ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int dim = RT == 16 ? d * 8 + (lane & 3) * 2 + (x & 1) : d * 16 + (lane >> 2) + 8 * (x >> 1);
                const int j = RT == 16 ? x >> 1 : x & 1;
                uint16_t raw;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(raw) : "r"(vs + tile_at(kw + key, dim >> 3) + (dim & 7) * 2));
                if (see[j] && finite16<BF16>(raw) != raw) A.o[d][x] = fmaf(p[j], from16<BF16>(raw), A.o[d][x]);
            }
    }
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int D, bool BF16, bool F32, int RT>
__global__ void __launch_bounds__(kAtThreads, SplitShape<D, RT>::PER_SM)
    attn_split_kernel(const AttnArgs P, const __grid_constant__ CUtensorMap pre_k, const __grid_constant__ CUtensorMap pre_v,
                      const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v) {
    using Sh = SplitShape<D, RT>;
    constexpr int NS = Sh::STAGES, TB = Sh::TILE, MR = Sh::MERGE_ROW, J = RT / 8;
    extern __shared__ __align__(128) uint8_t at_smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar[2 * NS];
    __shared__ int s_fail;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.x;
    const uint32_t full = smem_u32(s_bar), empty = full + 8 * NS;
    volatile int *fail = &s_fail;
    if (tid == 128) {
        s_fail = 0;
        for (int i = 0; i < NS; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 4);
        }
        fence_mbar_init();
    }
    // The tensor-memory kernel before this one lets it begin when all before itself is done: nothing to wait for then.
    const bool alone = !P.tc_pre && !P.tc_own;
    if (alone) griddep_wait();
    griddep_launch_dependents();
    const int nkv = P.own.n_kv, per_seq = nkv * P.mt_own;
    const int tp = P.mt_pre ? (P.prefix_len + kAtKeys - 1) / kAtKeys : 0;
    const long long line_pre = (long long)nkv * P.mt_pre * tp;
    long long first, end;
    int seq = 0, off = 0;
    if (!line_share<kAtThreads / 32>(P.own.n_seq, [&](int b) { return own_tiles(P, b); }, per_seq, line_pre, P.ctas, 1, first, end, seq, off)) {
        griddep_wait();
        return;
    }
    AttnAt at;
    if (first < line_pre) {
        at.seq = -1;
        at.base = at.keys = P.prefix_len;
        at.tiles = tp;
        const int u = (int)(first / tp);
        at.kvh = u / P.mt_pre;
        at.mt = u % P.mt_pre;
        at.tile = (int)(first % tp);
    } else {
        at.seq = seq;
        at.base = P.base[seq];
        at.keys = own_keys(P, seq);
        at.tiles = own_tiles(P, seq);
        const int in = (int)(first - line_pre - (long long)off * per_seq);
        const int u = in / at.tiles;
        at.kvh = u / P.mt_own;
        at.mt = u % P.mt_own;
        at.tile = in % at.tiles;
    }
    uint8_t *smem = at_smem_raw + ((1024 - (smem_u32(at_smem_raw) & 1023)) & 1023);
    const uint32_t ring = smem_u32(smem);
    __syncthreads();
    const int steps = (int)(end - first);
    if (warp == 4) {  // copies
        if (elect_one()) {
            int st = 0;
            uint32_t ph = 1;
            for (int s = 0; s < steps; ++s) {
                um_spin(empty + 8 * st, ph, fail);
                if (*fail) break;
                mbar_expect_tx(full + 8 * st, 2 * TB);
                const CUtensorMap *mk = at.seq < 0 ? &pre_k : &own_k, *mv = at.seq < 0 ? &pre_v : &own_v;
                const int t0 = at.tile * kAtKeys, sq = at.seq < 0 ? 0 : at.seq;
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
                    tma_load_4d(ring + st * 2 * TB + b * (kAtKeys * 128), mk, b * 64, t0, at.kvh, sq, full + 8 * st);
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
                    tma_load_4d(ring + st * 2 * TB + TB + b * (kAtKeys * 128), mv, b * 64, t0, at.kvh, sq, full + 8 * st);
                attn_step(P, at);
                if (++st == NS) {
                    st = 0;
                    ph ^= 1u;
                }
            }
        }
        __syncwarp();
    } else {
        float *merge = reinterpret_cast<float *>(smem + 2 * NS * TB);
        float2(*s_ml)[RT] = reinterpret_cast<float2(*)[RT]>(merge);  // the warps' statistics, before their outputs
        AttnAcc<D, RT> A;
        uint32_t qf[D / 16][RT / 4];
        bool fresh = true;
        int st = 0, M = 0, r0 = 0;
        uint32_t ph = 0;
        for (int s = 0; s < steps; ++s) {
            if (fresh) {  // a new (problem, row tile): its query vectors, empty statistics
                fresh = false;
                const int row0 = at.seq < 0 ? 0 : at.seq * P.rows;
                M = (at.seq < 0 ? P.S : P.rows) * P.G;
                r0 = at.mt * RT;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int r = r0 + (lane >> 2) + 8 * j;
                    const uint16_t *src = P.q + ((long long)(row0 + r / P.G) * P.H + at.kvh * P.G + r % P.G) * D + (lane & 3) * 2;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            qf[kk][j + J * e] = r < M ? *reinterpret_cast<const uint32_t *>(src + kk * 16 + e * 8) : 0u;
                }
#pragma unroll
                for (int d = 0; d < (int)(sizeof(A.o) / 16); ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) A.o[d][e] = 0.0f;
#pragma unroll
                for (int j = 0; j < J; ++j) A.m[j] = -INFINITY, A.l[j] = 0.0f;
                if (tid == 0 && at.tile == 0) P.cta_of[attn_unit(P, at)].x = c;
            }
            um_spin(full + 8 * st, ph, fail);
            attn_tile<D, BF16, F32, RT>(P, at, A, qf, ring + st * 2 * TB, ring + st * 2 * TB + TB, warp * 16, r0, M);
            __syncwarp();
            mbar_arrive_lane0(empty + 8 * st, lane);
            if (++st == NS) {
                st = 0;
                ph ^= 1u;
            }
            if (s + 1 == steps || at.tile + 1 == at.tiles) {  // one partial result: the four warps' added up in a fixed order
                const int unit = attn_unit(P, at);
                if (tid == 0 && at.tile + 1 == at.tiles) P.cta_of[unit].y = c;
                const long long row = ((long long)unit + c) * RT;
                consumer_sync();  // the last partial has been read
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    A.l[j] += __shfl_xor_sync(0xffffffffu, A.l[j], 1);
                    A.l[j] += __shfl_xor_sync(0xffffffffu, A.l[j], 2);
                    if ((lane & 3) == 0) s_ml[warp][(lane >> 2) + 8 * j] = make_float2(A.m[j], A.l[j]);
                }
                consumer_sync();
                float f[J];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int rr = (lane >> 2) + 8 * j;
                    float m = -INFINITY, l = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; ++w) m = fmaxf(m, s_ml[w][rr].x);
                    const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
                    for (int w = 0; w < 4; ++w) l += s_ml[w][rr].y * ex2(s_ml[w][rr].x - ms);
                    f[j] = ex2(A.m[j] - ms);
                    if (warp == 0 && (lane & 3) == 0 && r0 + rr < M) P.ml[row + rr] = make_float2(m, l);
                }
                consumer_sync();
                float g[2] = {f[0], f[J - 1]};
                if (RT == 8) {
                    g[0] = __shfl_sync(0xffffffffu, f[0], (lane & 3) * 8);
                    g[1] = __shfl_sync(0xffffffffu, f[0], (lane & 3) * 8 + 4);
                }
                for (int w = 0; w < 4; ++w) {
                    if (warp == w) {
#pragma unroll
                        for (int d = 0; d < (int)(sizeof(A.o) / 16); ++d)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int rr = RT == 16 ? (lane >> 2) + 8 * (e >> 1) : (lane & 3) * 2 + (e & 1);
                                const int dim = RT == 16 ? d * 8 + (lane & 3) * 2 + (e & 1) : d * 16 + (lane >> 2) + 8 * (e >> 1);
                                float *to = merge + rr * MR + dim;
                                const float v = A.o[d][e] * g[RT == 16 ? e >> 1 : e & 1];
                                *to = w ? *to + v : v;
                            }
                    }
                    consumer_sync();
                }
                const int have = min(RT, M - r0);
                for (int x = tid; x < have * (D / 4); x += 128) {
                    const int rr = x / (D / 4), ch = x % (D / 4);
                    *reinterpret_cast<float4 *>(P.part + (row + rr) * D + ch * 4) = *reinterpret_cast<const float4 *>(merge + rr * MR + ch * 4);
                }
                fresh = true;
            }
            attn_step(P, at);
        }
        if (tid == 0 && *fail) {
            report_error(P.err, kErrBarrierTimeout);
            const long long t0 = clock64();  // copies that are under way land before the shared memory is given back
            while (clock64() - t0 < 4000000LL) {
            }
        }
    }
    griddep_wait();  // the joining launch waits for this one alone, and needs the tensor-memory kernel's results too
}

// The partials of a row vector lie in up to six runs of rows of part / ml: `n` rows, `stride` apart, from row `at` on.
// Lane j < 6 of a warp holds run j.
struct AttnRun {
    long long at;
    int stride, n;
};
// Run j of row vector r (within its sequence) of a (sequence, kv head), but for the CTAs that share its unit: the prefix's and
// the own slots' from the split kernel (0, 1), the same from the tensor-memory kernel, each in up to two halves (2 to 5).  It
// needs no other launch's results.
struct AttnRunOf {
    int unit, row, stride;
    bool there, tc;
};
__device__ __forceinline__ AttnRunOf attn_run_of(const AttnArgs &P, int j, int seq, int kvh, int r, int rt) {
    const int nkv = P.own.n_kv, rp = seq * P.rows * P.G + r;
    const bool own = j == 1 || j >= 4;
    const int q = own ? r : rp;
    AttnRunOf R;
    R.tc = j >= 2;
    int t, from;  // rows of a unit that row vectors are dealt out by, first unit of the kv head
    if (!R.tc) {
        t = R.stride = rt;
        R.there = own ? own_tiles(P, seq) > 0 : P.mt_pre > 0;
        from = own ? nkv * P.mt_pre + (seq * nkv + kvh) * P.mt_own : kvh * P.mt_pre;
    } else {
        const int two = own ? P.tc2_own : P.tc2_pre;
        R.stride = P.tc_rows;
        t = two ? 128 : P.tc_rows;
        R.there = (own ? P.tc_own && own_keys(P, seq) > 0 : P.tc_pre) && (two || !(j & 1));
        from = own ? nkv * P.tcm_pre + (seq * nkv + kvh) * P.tcm_own : kvh * P.tcm_pre;
    }
    R.there = R.there && j < 6;
    const int mt = (int)((unsigned)q / (unsigned)t);
    R.unit = from + mt;
    R.row = q - mt * t + (R.tc && (j & 1) ? 128 : 0);
    return R;
}
__device__ __forceinline__ AttnRun attn_run(const AttnArgs &P, const AttnRunOf &of) {
    AttnRun R{0, of.stride, 0};
    if (of.there) {
        const int2 ends = (of.tc ? P.tc_cta_of : P.cta_of)[of.unit];
        R.n = ends.y - ends.x + 1;
        R.at = ((long long)of.unit + ends.x) * of.stride + of.row + (of.tc ? P.tc_row0 : 0);
    }
    return R;
}
// Row of part / ml of partial j, counted over all runs.
__device__ __forceinline__ long long attn_partial(const AttnRun &run, int j) {
    int in = 0, off = 0;
#pragma unroll
    for (int k = 0; k < 6; ++k) {
        const int n = __shfl_sync(0xffffffffu, run.n, k);
        if (j >= 0 && j < n) {
            in = k;
            off = j;
        }
        j -= n;
    }
    const long long at = __shfl_sync(0xffffffffu, run.at, in);
    return at + (long long)off * __shfl_sync(0xffffffffu, run.stride, in);
}
// What the statistics of all partials say: maximum and sum; and each lane's place among the first 32, with its maximum.
struct AttnRow {
    long long at;
    int n;
    float m, l, at_m;
};
__device__ __forceinline__ AttnRow attn_row(const AttnArgs &P, const AttnRun &run, int lane) {
    AttnRow R;
    R.n = __reduce_add_sync(0xffffffffu, lane < 6 ? run.n : 0);
    float m = -INFINITY, l = 0.0f;
    for (int j0 = 0; j0 < R.n || j0 == 0; j0 += 32) {
        const long long at = attn_partial(run, j0 + lane);
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (j0 + lane < R.n) ml = P.ml[at];
        if (j0 == 0) {
            R.at = at;
            R.at_m = ml.x;
        }
        const float to = fmaxf(m, ml.x);
        if (to != -INFINITY) {
            l = l * ex2(m - to) + ml.y * ex2(ml.x - to);
            m = to;
        } else {
            l += ml.y;  // zero, or NaN
        }
    }
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.0f;
    l *= ex2(m - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    R.m = top;
    R.l = l;
    return R;
}

// Adds the weights 2^(x - m) / l of four slots to their sums.
__device__ __forceinline__ void attn_weigh(float (&sum)[4], const float4 &x, const float2 &st) {
    if (x.x != -INFINITY) sum[0] = fmaf(ex2(x.x - st.x), st.y, sum[0]);
    if (x.y != -INFINITY) sum[1] = fmaf(ex2(x.y - st.x), st.y, sum[1]);
    if (x.z != -INFINITY) sum[2] = fmaf(ex2(x.z - st.x), st.y, sum[2]);
    if (x.w != -INFINITY) sum[3] = fmaf(ex2(x.w - st.x), st.y, sum[3]);
}

// Joins the partials.  The first `row_ctas` CTAs take 4 / WPR row vectors each, WPR warps to one (4 where there are too few
// row vectors to fill the device with a warp each: below 16 an SM.  A call of 16, 24, 36 and 38 rows x 64 heads behind 8192 keys
// takes 29.3, 37.2, 54.1 and 54.5 us with four warps, 34.1, 37.8, 51.1 and 51.3 with one; the last two lie on either side
// of the border); with acc and up to kAtMany row vectors a problem, further CTAs take 1024 slots of one
// (sequence, kv head) each.  What bounds it is a chain of latencies (CTAs of a unit, statistics, partials), so all that does
// not hang on the launches before comes ahead of the wait for them, and eight partials of a warp are under way together.
template <int D, bool BF16, int WPR>
__global__ void __launch_bounds__(kAtCombine) attn_join_kernel(const AttnArgs P, int rt, int row_ctas, int chunks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x < (unsigned)row_ctas) {
        constexpr int E = D / 32;
        __shared__ float s_o[WPR][WPR == 1 ? 1 : D];
        const unsigned u = blockIdx.x * (4 / WPR) + warp / WPR;
        const int sub = warp % WPR;
        // lengths came before the launches that this one waits for
        const bool mine = u < (unsigned)(P.S * P.H);
        const unsigned row = u / (unsigned)P.H, h = u - row * P.H, seq = row / (unsigned)P.rows, kvh = h / (unsigned)P.G;
        const bool none = !mine || P.base[seq] < 0;
        AttnRunOf of{};
        if (!none) of = attn_run_of(P, lane, seq, kvh, (row - seq * P.rows) * P.G + (h - kvh * P.G), rt);
        griddep_wait();
        griddep_launch_dependents();
        if (none) return;
        const AttnRun run = attn_run(P, of);
        const AttnRow R = attn_row(P, run, lane);
        float o[E] = {};
        for (int j0 = 0; j0 < R.n; j0 += 32) {
            const long long mine = j0 ? attn_partial(run, j0 + lane) : R.at;
            const float w = j0 + lane < R.n ? ex2((j0 ? P.ml[mine].x : R.at_m) - R.m) : 0.0f;
            const int n = min(32, R.n - j0);
            constexpr int V = E < 4 ? 2 : 4, B = 8;  // floats of a load, partials under way together
            for (int i0 = sub; i0 < n; i0 += B * WPR) {
                float x[B][E];
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const int i = i0 + k * WPR;
                    const float *src = P.part + __shfl_sync(0xffffffffu, mine, i & 31) * D + lane * E;
#pragma unroll
                    for (int e = 0; e < E; e += V) {
                        if (V == 2) {
                            const float2 v = i < n ? *reinterpret_cast<const float2 *>(src + e) : make_float2(0.0f, 0.0f);
                            x[k][e] = v.x, x[k][e + 1] = v.y;
                        } else {
                            const float4 v = i < n ? *reinterpret_cast<const float4 *>(src + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            x[k][e] = v.x, x[k][e + 1] = v.y, x[k][(e + 2) % E] = v.z, x[k][(e + 3) % E] = v.w;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < B; ++k) {
                    const int i = i0 + k * WPR;
                    const float f = __shfl_sync(0xffffffffu, w, i & 31);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = fmaf(x[k][e], i < n ? f : 0.0f, o[e]);
                }
            }
        }
        if (WPR > 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) s_o[sub][WPR == 1 ? 0 : lane * E + e] = o[e];
            __syncthreads();
            if (sub) return;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int d = WPR == 1 ? 0 : lane * E + e;
                o[e] = (s_o[0][d] + s_o[1 % WPR][d]) + (s_o[2 % WPR][d] + s_o[3 % WPR][d]);
            }
        }
        const float inv = R.l == 0.0f ? 0.0f : 1.0f / R.l;
        if (P.stats && lane == 0) P.stats[u] = make_float2(R.m - kAtLift<BF16>, inv);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= inv;
        const long long to = (long long)u * D + lane * E;
        if (P.out_f32) {
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<float2 *>(static_cast<float *>(P.out) + to + e) = make_float2(o[e], o[e + 1]);
        } else {
#pragma unroll
            for (int e = 0; e < E; e += 2)
                *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(P.out) + to + e) = pack16<BF16>(o[e], o[e + 1]);
        }
        return;
    }
    // acc[slot] += sum over the group's row vectors of 2^(x - m) / l
    griddep_wait();
    griddep_launch_dependents();
    const int u = blockIdx.x - row_ctas, g = u / chunks, chunk = u % chunks;
    const int seq = g / P.own.n_kv, kvh = g % P.own.n_kv;
    const int keys = own_keys(P, seq);
    if (chunk * kAtChunk >= keys) return;
    constexpr int C = kAtChunk / kAtCombine;
    __shared__ float2 s_row[kAtMany];  // m and 1 / l of the row vectors
    const int M = P.rows * P.G, t0 = chunk * kAtChunk + threadIdx.x;
    for (int r = warp; r < M; r += 4) {
        const AttnRow R = attn_row(P, attn_run(P, attn_run_of(P, lane, seq, kvh, r, rt)), lane);
        if (lane == 0) s_row[r] = make_float2(R.m - kAtLift<BF16>, R.l == 0.0f ? 0.0f : 1.0f / R.l);
    }
    __syncthreads();
    float sum[C] = {};
    const float *x = P.scores + (long long)g * M * P.own.cap + t0;
    for (int r = 0; r < M; ++r, x += P.own.cap) {
        const float2 st = s_row[r];
        float w[C];
#pragma unroll
        for (int j = 0; j < C; ++j) w[j] = t0 + j * kAtCombine < keys ? x[j * kAtCombine] : -INFINITY;
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (w[j] != -INFINITY) sum[j] = fmaf(ex2(w[j] - st.x), st.y, sum[j]);
    }
    float *acc = P.own.acc + (long long)g * P.own.cap + t0;
#pragma unroll
    for (int j = 0; j < C; ++j)
        if (t0 + j * kAtCombine < keys) acc[j * kAtCombine] += sum[j];
}

// The same for problems of many row vectors: a warp takes four slots of one (sequence, kv head), its lanes the row vectors.
__global__ void __launch_bounds__(256) attn_acc_kernel(const AttnArgs P, int chunks) {
    griddep_wait();
    griddep_launch_dependents();
    const int g = blockIdx.x / chunks, q = blockIdx.x % chunks * 8 + (threadIdx.x >> 5), seq = g / P.own.n_kv, kvh = g % P.own.n_kv;
    const int keys = own_keys(P, seq), M = P.rows * P.G, lane = threadIdx.x & 31;
    if (4 * q >= keys) return;
    const float2 *stats = P.stats + (long long)seq * P.rows * P.H + kvh * P.G;
    float sum[4] = {};
#pragma unroll 4
    for (int r = lane; r < M; r += 32)
        attn_weigh(sum, *reinterpret_cast<const float4 *>(score_at(P, g, q, M, r)), stats[(long long)(r / P.G) * P.H + r % P.G]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
    const int t = 4 * q + lane;
    if (lane < 4 && t < keys) P.own.acc[(long long)g * P.own.cap + t] += lane == 0 ? sum[0] : lane == 1 ? sum[1] : lane == 2 ? sum[2] : sum[3];
}

}  // namespace pgb
