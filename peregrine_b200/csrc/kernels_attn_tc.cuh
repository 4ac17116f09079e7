// Attention of problems with many row vectors (a prefix under a whole batch, a prompt chunk) on the tensor-memory units.
//
// A CTA holds two tiles of 128 query vectors in shared memory and streams tiles of keys and values past them:
//     S = Q K^T (tensor memory) -> weights 2^(x - m), written over S as the A operand -> O += P V (tensor memory)
// Two threads own a row (its TMEM lane), 32 columns of a tile each: with one, two warps a scheduler form the weights and hide
// little of each other's latencies (53.5 us instead of 51.7 for the call below).  The two row tiles
// alternate: while one's weights are formed the tensor unit works for the other.  A step of 64 keys x 256 rows (D = 128) takes the
// tensor unit 1280 cycles at the least (a 64-column product of the scores reads its operands from shared memory for 48 cycles and
// multiplies for 32; the second product 64) and the exponential unit (16 a cycle) 1024, so neither can wait for the other; S has
// two buffers where they fit, so that the next scores are there when a tile's weights are done.  O is rescaled only when a
// row's maximum has grown by 2^8 since it was last set: m only has to keep weights in range, and cancels in O / l.  With at most 128 row vectors both tiles hold the same ones and the key tiles go to them in turn.  D = 256 has
// no room for a second O: there one tile alternates between two S.
//
// Measured: 32 rows x 64 heads behind 32768 keys (8 key heads of 128, bf16 out, keys from HBM) 46 us, 747 TFLOP/s of the 1669
// that cuBLAS reaches.  A CTA's 43 us (the slowest's 45): 2.1 until its place on the line is known, 3.1 until the first scores
// are there, 33.5 for 28 steps, 3.2 until its partial result is written, 1.1 until the last warp of it is done.  The first step takes
// 2.8 us (the second tile is asked for when the query vectors are there), the others 1.10 us, 1950 cycles at 1.77 GHz: the
// issuing thread waits about 270 of them for weights and stands in the tensor unit's full queue for nearly all others; a
// step's keys and values are there when it asks (2.9 TB/s).
//
// Only the last tiles of a problem have keys that some row does not see; there, S is masked after it was read, and what the
// values of such keys may hold is taken out of the tile in shared memory before the product (0 x inf is not 0).  Work is
// dealt out as in kernels_attn.cuh: one line of key tiles, equal parts.
#pragma once
#include "kernels_attn.cuh"

namespace pgb {

// Tiles that a change of the problem costs a CTA (query vectors, first and last tile, its partial result): on the line every
// (problem, row tile) begins with so many empty ones.  With 4, 8 and 16: 5 drafts of 8 rows (28 heads of 64) 23.7, 24.8 and 26.5 us,
// 64 x 8 rows (32 heads of 128) over 300 slots 52.5, 54.6 and 59.1, over 2000 slots 119.9, 117.8 and 124.2, the call above the same.
constexpr int kTcEmpty = 8;
// Tiles (empty ones too) of a CTA at least.  With 1, 4 and 8: 8 rows over 3000 slots (4 key heads of 128) 18.0, 16.9 and 21.6 us, 64 x 64 heads
// behind 32768 keys 87.8, 86.7 and 86.8; but 64 rows over 1500 slots (4 key heads of 128) 17.1, 23.5 and 31.0.
constexpr int kTcLeast = 4;

template <int D, bool BF16, bool F32>
struct TcShape {
    static constexpr int TILES = D == 256 ? 1 : 2;  // row tiles of a CTA, 8 softmax warps each
    static constexpr int TERMS = kAtTerms<BF16, F32>;
    // S buffers of a row tile, and their columns.  32 keys of weights take 16 columns a term; three terms outgrow the S that
    // they replace, which then sits in the upper half of a larger buffer.
    static constexpr int BUFS = D == 256 || TERMS < 3 ? 2 : 1;
    static constexpr int BUF_COLS = D < 256 && TERMS < 3 ? 64 : 128;
    static constexpr int S_COL = TERMS == 3 ? 64 : 0;
    static constexpr int O_COL = 256;
    static_assert(TILES * BUFS * BUF_COLS == 256 && O_COL + TILES * D <= 512, "columns");
    static constexpr int N = kTcKeys;
    static constexpr int Q_BYTES = 128 * D * 2, TILE_BYTES = N * D * 2;
    static constexpr int FIT = (232448 - 5120 - TILES * Q_BYTES) / TILE_BYTES;
    static constexpr int SLOTS = FIT > 12 ? 12 : FIT;
    static constexpr int SMEM = 1024 + TILES * Q_BYTES + SLOTS * TILE_BYTES;
    static constexpr int THREADS = TILES * 256 + 64;  // softmax, copies, matrix instructions
    static constexpr int ROWS = TILES * 128;
};

// A place on the line; tiles and tile count the empty ones.
struct TcAt {
    int seq, kvh, mt, tile, tiles;
};
__device__ __forceinline__ int tc_tiles(const AttnArgs &P, int b) {
    const int n = P.tc_own ? (own_keys(P, b) + kTcKeys - 1) / kTcKeys : 0;
    return n ? n + kTcEmpty : 0;
}
// The key tiles [t0, t0 + n) of the place's (problem, row tile) that lie in the next `left` tiles of the line; takes them off.
__device__ __forceinline__ int tc_segment(const TcAt &a, int &left, int &t0) {
    const int v = min(left, a.tiles - a.tile), t1 = a.tile + v - kTcEmpty;
    left -= v;
    t0 = max(a.tile - kTcEmpty, 0);
    return max(t1 - t0, 0);
}
// Moves to the next (problem, row tile) with tiles.
__device__ __forceinline__ void tc_next(const AttnArgs &P, TcAt &a) {
    a.tile = 0;
    if (++a.mt < (a.seq < 0 ? P.tcm_pre : P.tcm_own)) return;
    a.mt = 0;
    if (++a.kvh < P.own.n_kv) return;
    a.kvh = 0;
    do {
        if (++a.seq >= P.own.n_seq) {
            a.seq = P.own.n_seq - 1;
            return;
        }
        a.tiles = tc_tiles(P, a.seq);
    } while (a.tiles == 0);
}

__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo) {  // 128-byte swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tile_sync(int w) { asm volatile("bar.sync %0, 256;" ::"r"(9 + w) : "memory"); }  // the warps of a row tile
__device__ __forceinline__ bool rows_any(int w, int q, bool v) {  // the same with a vote
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %2, 0;\n\tbar.red.or.pred p, %1, 64, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(r)
                 : "r"(1 + w * 4 + q), "r"((uint32_t)v)
                 : "memory");
    return r != 0;
}
__device__ __forceinline__ void rows_sync(int w, int q) { asm volatile("bar.sync %0, 64;" ::"r"(1 + w * 4 + q) : "memory"); }  // the two of 32 rows
// Swizzle of 16-byte pieces in rows of `pieces` (4 or 8) of them: eight neighbouring rows or pieces meet all banks.
__device__ __forceinline__ int turn_at(int row, int pieces) { return pieces == 8 ? row & 7 : (row >> 1) & 3; }
__device__ __forceinline__ uint32_t low32(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }  // n low bits
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Pairs of fp32 values, an operation on both at once.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^y of both halves for finite y: 2^n 2^f with n the nearest whole number, found by adding 1.5 x 2^23, and the Taylor sum of
// e^(f ln 2), |f| <= 1/2, to the power DEG: off by (ln 2 / 2)^(DEG + 1) / (DEG + 1)!, 4.2e-5 or 2.4e-6 for 4, 5.
// Below 2^-126 the result stays there.
template <int DEG>
__device__ __forceinline__ void exp2_poly(uint64_t y, float &lo, float &hi) {
    constexpr float kC[6] = {1.0f, 0.69314718056f, 0.24022650696f, 0.05550410866f, 0.00961812911f, 0.00133335581f};  // ln(2)^k / k!
    float a, b;
    unpack2(y, a, b);
    a = fmaxf(a, -126.0f);
    b = fmaxf(b, -126.0f);
    y = pack2(a, b);
    const uint64_t t = add2(y, pack2(12582912.0f, 12582912.0f));
    const uint64_t f = fma2(add2(t, pack2(-12582912.0f, -12582912.0f)), pack2(-1.0f, -1.0f), y);
    uint64_t p = pack2(kC[DEG], kC[DEG]);
#pragma unroll
    for (int k = DEG - 1; k >= 0; --k) p = fma2(p, f, pack2(kC[k], kC[k]));
    float ta, tb;
    unpack2(t, ta, tb);
    unpack2(p, a, b);
    lo = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23));
    hi = __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23));
}
// `i`-th user of a ring of n: its place and the parity of its turn.
template <int n>
struct RingAt {
    int i = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next(int k) {  // k < n
        i += k;
        if (i >= n) {
            i -= n;
            ph ^= 1u;
        }
    }
    __device__ __forceinline__ void skip(int k) {
        i += k;
        while (i >= n) {
            i -= n;
            ph ^= 1u;
        }
    }
};

template <int D, bool BF16, bool F32>
__global__ void __launch_bounds__(TcShape<D, BF16, F32>::THREADS, 1)
    attn_tc_kernel(const AttnArgs P, const __grid_constant__ CUtensorMap pre_k, const __grid_constant__ CUtensorMap pre_v,
                   const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v) {
    using T = TcShape<D, BF16, F32>;
    constexpr int N = T::N, DB = D / 64;
    extern __shared__ __align__(128) uint8_t tc_smem_raw[];
    __shared__ __align__(8) unsigned long long s_bar[2 * T::SLOTS + 3 * T::TILES + 2 * T::TILES * T::BUFS];
    __shared__ uint32_t s_tmem;
    __shared__ float s_top[2][T::TILES][2][128];  // a row's two maxima, by turns
    __shared__ int s_fail;
    // New slots in which infinite or NaN values were met, a bit each.  Only a hint of where to look again: bits stay.
    __shared__ unsigned s_odd[2];
    const int tid = threadIdx.x, warp = tid >> 5, c = blockIdx.x;
    uint8_t *base = tc_smem_raw + ((1024 - (smem_u32(tc_smem_raw) & 1023)) & 1023);
    const uint32_t q_s = smem_u32(base), ring_s = q_s + T::TILES * T::Q_BYTES;
    const uint32_t full = smem_u32(s_bar), empty = full + 8 * T::SLOTS, qfull = empty + 8 * T::SLOTS, odone = qfull + 8 * T::TILES,
                   sfull = odone + 8 * T::TILES, pfull = sfull + 8 * T::TILES * T::BUFS,
                   pvdone = pfull + 8 * T::TILES * T::BUFS;
    volatile int *fail = &s_fail;
    constexpr int kProducer = T::TILES * 8, kIssuer = kProducer + 1;
    if (tid == 0) {
        s_fail = 0;
        s_odd[0] = s_odd[1] = 0;
        for (int i = 0; i < 2 * T::SLOTS; ++i) mbar_init(full + 8 * i, 1);
        for (int i = 0; i < T::TILES; ++i) {
            mbar_init(qfull + 8 * i, 8);
            mbar_init(odone + 8 * i, 1);
            mbar_init(pvdone + 8 * i, 1);
        }
        for (int i = 0; i < T::TILES * T::BUFS; ++i) {
            mbar_init(sfull + 8 * i, 1);
            mbar_init(pfull + 8 * i, 8);
        }
        fence_mbar_init();
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = s_tmem;
    griddep_wait();
    griddep_launch_dependents();  // (now, when all before this launch is done: the next one does not wait for it)
    const int nkv = P.own.n_kv, per_seq = nkv * P.tcm_own, tp = P.tc_pre ? (P.prefix_len + N - 1) / N + kTcEmpty : 0;
    const long long line_pre = (long long)nkv * P.tcm_pre * tp;
    long long first = 0, end = 0;
    int seq = 0, off = 0;
    if (!line_share<T::THREADS / 32>(P.tc_own ? P.own.n_seq : 0, [&](int b) { return tc_tiles(P, b); }, per_seq, line_pre, P.tc_ctas, kTcLeast, first, end, seq,
                                     off))
        first = end = 0;
    TcAt at;
    if (first == end) {
        at = TcAt{0, 0, 0, 0, 0};
    } else if (first < line_pre) {
        const int u = (int)(first / tp);
        at = TcAt{-1, u / P.tcm_pre, u % P.tcm_pre, (int)(first % tp), tp};
    } else {
        const int tiles = tc_tiles(P, seq);
        const long long in = first - line_pre - (long long)off * per_seq;
        const int u = (int)(in / tiles);
        at = TcAt{seq, u / P.tcm_own, u % P.tcm_own, (int)(in % tiles), tiles};
    }
    int left = (int)(end - first);
    if (warp == kProducer) {
        // ================================================================ copies: K and V of a tile in boxes of 64 keys x 64 dims
        if (elect_one()) {
            RingAt<T::SLOTS> r;
            bool begun = false;
            while (left > 0 && !*fail) {
                int t0;
                const int n = tc_segment(at, left, t0), s = at.seq < 0 ? 0 : at.seq;
                const CUtensorMap *mk = at.seq < 0 ? &pre_k : &own_k, *mv = at.seq < 0 ? &pre_v : &own_v;
                for (int j = 0; j < n && !*fail; ++j)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        um_spin(empty + 8 * r.i, r.ph ^ 1u, fail);
                        if (*fail) break;
                        mbar_expect_tx(full + 8 * r.i, T::TILE_BYTES);
#pragma unroll
                        for (int b = 0; b < DB; ++b)
                            tma_load_4d(ring_s + r.i * T::TILE_BYTES + b * (N * 128), v ? mv : mk, b * 64, (t0 + j) * N, at.kvh, s, full + 8 * r.i);
                        r.next(1);
                        if (!begun && v) {
                            // The query vectors' loads must not queue behind a ring full of tiles.  (With three tiles to come
                            // the barrier stays in this phase until they do.)
                            begun = true;
                            if (n > 2) um_spin(qfull, 0u, fail);
                        }
                    }
                tc_next(P, at);
            }
        }
    } else if (warp == kIssuer) {
        // ================================================================ matrix instructions
        if (elect_one()) {
            constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t kIdescS = (1u << 4) | kType | ((uint32_t)(N >> 3) << 17) | (8u << 24);
            constexpr uint32_t kIdescO = (1u << 4) | kType | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);  // V: dims contiguous
            RingAt<T::SLOTS> seg;  // the ring place of the segment's first K
            uint32_t qph = 0, pph = 0;
            for (; left > 0 && !*fail; tc_next(P, at)) {
                int t0;
                const int n = tc_segment(at, left, t0);
                const int two = T::TILES == 2 && (at.seq < 0 ? P.tc2_pre : P.tc2_own);
                // tile i of row tile w is key tile `i` of the segment, or 2 i + w when they take turns
                const int step = two ? 4 : 2;
                int count[T::TILES], most = 0;
                RingAt<T::SLOTS> kp[T::TILES], vp[T::TILES];  // of the row tiles' next K and V
#pragma unroll
                for (int w = 0; w < T::TILES; ++w) {
                    count[w] = two ? (n + 1 - w) >> 1 : n;
                    most = max(most, count[w]);
                    kp[w] = seg;
                    if (two && w) kp[w].next(2);
                    vp[w] = kp[w];
                    vp[w].next(1);
                }
                auto scores = [&](int w, int i) {
                    const RingAt<T::SLOTS> r = kp[w];
                    kp[w].next(step);
                    if (i == 0) um_spin(qfull + 8 * w, (qph >> w) & 1u, fail);
                    if (w == 0 || two) um_spin(full + 8 * r.i, r.ph, fail);
                    tmem_fence_after();
                    const uint32_t d = tmem + (w * T::BUFS + i % T::BUFS) * T::BUF_COLS + T::S_COL;
                    const uint64_t qd = desc_sw128(q_s + w * T::Q_BYTES, 16), kd = desc_sw128(ring_s + r.i * T::TILE_BYTES, 16);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_f16_ss(d, qd + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2, kd + (k >> 2) * (N * 128 / 16) + (k & 3) * 2, kIdescS, k > 0);
                    if (w == T::TILES - 1 || two) umma_commit(empty + 8 * r.i);
                    umma_commit(sfull + 8 * (w * T::BUFS + i % T::BUFS));
                };
#pragma unroll
                for (int b = 0; b < T::BUFS; ++b)
#pragma unroll
                    for (int w = 0; w < T::TILES; ++w)
                        if (b < count[w]) scores(w, b);
#pragma unroll
                for (int w = 0; w < T::TILES; ++w)
                    if (count[w]) qph ^= 1u << w;
                for (int i = 0; i < most && !*fail; ++i)
#pragma unroll
                    for (int w = 0; w < T::TILES; ++w) {
                        if (i >= count[w]) continue;
                        const RingAt<T::SLOTS> r = vp[w];
                        vp[w].next(step);
                        const int bi = i % T::BUFS, buf = w * T::BUFS + bi;
                        um_spin(pfull + 8 * buf, (pph >> buf) & 1u, fail);
                        pph ^= 1u << buf;
                        if (w == 0 || two) um_spin(full + 8 * r.i, r.ph, fail);
                        tmem_fence_after();
                        const uint64_t vd = desc_sw128(ring_s + r.i * T::TILE_BYTES, N * 128);
                        const uint32_t pa = tmem + buf * T::BUF_COLS;
#pragma unroll
                        for (int k = 0; k < N / 16; ++k)
#pragma unroll
                            for (int t = 0; t < T::TERMS; ++t)
                                umma_f16_ts(tmem + T::O_COL + w * D, pa + (k >> 1) * (16 * T::TERMS) + t * 16 + (k & 1) * 8, vd + k * (2048 / 16),
                                            kIdescO, i > 0 || k > 0 || t > 0);
                        if (w == T::TILES - 1 || two) umma_commit(empty + 8 * r.i);
                        if (i + 1 == count[w]) {
                            umma_commit(odone + 8 * w);
                        } else {
                            if (T::BUFS > 1) umma_commit(pvdone + 8 * w);
                            if (i + T::BUFS < count[w]) scores(w, i + T::BUFS);
                        }
                    }
                seg.skip(2 * n % T::SLOTS);
                if ((2 * n / T::SLOTS) & 1) seg.ph ^= 1u;
            }
        }
    } else {
        // ================================================================ softmax: half a row of row tile w per thread
        const int w = warp >> 3, hf = (warp >> 2) & 1, lane = tid & 31, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 TMEM lanes
        const uint32_t flip = P.scale2 < 0.0f ? 0x80008000u : 0u;  // the sign of the scale goes into Q: scores only need a positive one
        const float scale = fabsf(P.scale2);
        int turn = 0;
        RingAt<T::SLOTS> ring;  // the ring place of the segment's first K
        uint32_t sph[T::BUFS] = {}, oph = 0, pvph = 1;  // pvph: parity of the product before this tile's (the segment's last one is told by odone)
        for (; left > 0; tc_next(P, at)) {
            int t0;
            const int n = tc_segment(at, left, t0);
            if (n == 0) continue;  // empty tiles alone
            const int two = T::TILES == 2 && (at.seq < 0 ? P.tc2_pre : P.tc2_own);
            const int mine = two ? (n + 1 - w) >> 1 : n;
            const int M = (at.seq < 0 ? P.S : P.rows) * P.G, row0 = at.seq < 0 ? 0 : at.seq * P.rows;
            const int r = two ? at.mt * 128 + row : at.mt * T::ROWS + w * 128 + row;
            // keys below `seen` are seen by every row, new slots from `fresh` on by the row's bits, none from `keys` on
            const int fresh = at.seq < 0 ? P.prefix_len : P.base[at.seq], keys = at.seq < 0 ? P.prefix_len : own_keys(P, at.seq);
            const int seen = min(fresh, keys);
            const unsigned long long bits = at.seq >= 0 && r < M ? row_mask(P, at.seq * P.rows + r / P.G, r / P.G) : 0;
            float m = -INFINITY, l = 0.0f;
            if (mine) {
                // D / 8 lanes read a row together; a warp brings 16 of its 32 rows
                constexpr int LPR = D / 8, RPI = 32 / LPR, B = 16 / RPI;  // loads under way together
                const int ch = lane % LPR, rl = (row & ~31) + hf * 16 + lane / LPR;
                uint8_t *to = base + w * T::Q_BYTES + (ch >> 3) * (128 * 128);
                int q = r - row + rl, div = q / P.G, rem = q - div * P.G;  // row vector, its row and head
                const uint16_t *src = P.q + ((long long)row0 * P.H + at.kvh * P.G) * D + ch * 8;
#pragma unroll
                for (int i0 = 0; i0 < 16 / RPI; i0 += B) {
                    uint4 v[B];
#pragma unroll
                    for (int e = 0; e < B; ++e) {
                        v[e] = make_uint4(0, 0, 0, 0);
                        if (q < M) v[e] = *reinterpret_cast<const uint4 *>(src + ((long long)div * P.H + rem) * D);
                        q += RPI;
                        for (rem += RPI; rem >= P.G; ++div) rem -= P.G;
                    }
#pragma unroll
                    for (int e = 0; e < B; ++e) {
                        const int k = rl + (i0 + e) * RPI;
                        v[e].x ^= flip, v[e].y ^= flip, v[e].z ^= flip, v[e].w ^= flip;
                        *reinterpret_cast<uint4 *>(to + k * 128 + (((ch & 7) ^ (k & 7)) << 4)) = v[e];
                    }
                }
                fence_proxy_async();
                __syncwarp();
                mbar_arrive_lane0(qfull + 8 * w, lane);
            }
            for (int i = 0; i < mine; ++i) {
                const int bi = i % T::BUFS, buf = w * T::BUFS + bi;
                const uint32_t region = tmem + lanes + buf * T::BUF_COLS;
                um_spin(sfull + 8 * buf, sph[bi], fail);
                sph[bi] ^= 1u;
                tmem_fence_after();
                float s[32];
                tmem_ld32(region + T::S_COL + hf * 32, s);
                tmem_wait_ld32(s);
                const int j = two ? 2 * i + w : i, k0 = (t0 + j) * N, c0 = k0 + hf * 32;  // the tile's first key, this thread's
                const bool open = k0 + N <= seen;
                uint32_t see = 0xffffffffu;
                if (!open) {
                    const int d = c0 - fresh;
                    const unsigned long long late = d >= 64 || d <= -32 ? 0ull : d >= 0 ? bits >> d : bits << -d;
                    see = (low32(seen - c0) | (uint32_t)late) & low32(keys - c0);
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[e] = (see >> e) & 1u ? s[e] : -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int e = 4; e < 28; e += 8)
#pragma unroll
                    for (int f = 0; f < 4; ++f) mx[f] = max_nan(mx[f], s[e + f], s[e + 4 + f]);
                float top = max_nan(max_nan(max_nan(mx[0], mx[1], s[28]), max_nan(mx[2], mx[3], s[29])), s[30], s[31]);
                top = see ? top * scale : -INFINITY;
                // The usual tile needs no more than the two threads of every row to agree that it is one: no mask, no NaN, no
                // infinity, and no maximum that has grown too far.  (They have both read S then: weights may replace any of it.)
                if (i) pvph ^= 1u;
                bool plain = true, grown = false;
                if (rows_any(w, warp & 3, i == 0 || !(open && top <= m + kAtLag))) {
                    s_top[turn][w][hf][row] = top;
                    rows_sync(w, warp & 3);
                    top = max_nan(top, s_top[turn][w][hf ^ 1][row]);
                    turn ^= 1;
                    plain = __all_sync(0xffffffffu, open && top < INFINITY);
                    if (i == 0)
                        m = top;
                    else
                        grown = __any_sync(0xffffffffu, top > m + kAtLag);
                }
                if (grown) {
                    // O of this row tile is at rest: the product before was committed with these scores, or is waited for
                    if (T::BUFS > 1) {
                        um_spin(pvdone + 8 * w, pvph, fail);
                        tmem_fence_after();
                    }
                    const float to = top > m + kAtLag ? top : m;
                    const float f = to == m ? 1.0f : ex2(m - to);
                    m = to;
                    l *= f;
#pragma unroll 1
                    for (int d = hf * (D / 2); d < (hf + 1) * (D / 2); d += 32) {
                        float o[32];
                        tmem_ld32(tmem + lanes + T::O_COL + w * D + d, o);
                        tmem_wait_ld32(o);
                        uint32_t u[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[h * 16 + e] * f);
                            tmem_st16(tmem + lanes + T::O_COL + w * D + d + h * 16, u);
                        }
                    }
                }
                if (P.scores && at.seq >= 0 && r < M) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float x[4];
#pragma unroll
                        for (int f = 0; f < 4; ++f) x[f] = (see >> (e + f)) & 1u ? s[e + f] * scale : -INFINITY;
                        if (c0 + e < keys)
                            *reinterpret_cast<float4 *>(score_at(P, at.seq * nkv + at.kvh, (c0 + e) >> 2, M, r)) = make_float4(x[0], x[1], x[2], x[3]);
                    }
                }
                if (!open && at.seq >= 0) {
                    // values of slots that are not seen by all: zeros for those never stored, and for what is not finite (rows
                    // that do see such a value add it when the partial result is written)
                    RingAt<T::SLOTS> at_v = ring;
                    at_v.skip(2 * j + 1);
                    um_spin(full + 8 * at_v.i, at_v.ph, fail);
                    uint8_t *vt = base + (ring_s - q_s) + at_v.i * T::TILE_BYTES;
                    for (int x = tid & 255; x < N * (D / 8); x += 256) {
                        const int key = x / (D / 8), ch = x % (D / 8);
                        if (k0 + key < seen) continue;
                        uint4 *at_x = reinterpret_cast<uint4 *>(vt + (ch >> 3) * (N * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (k0 + key < keys) {
                            const uint4 o = *at_x;
                            v = make_uint4(finite16<BF16>(o.x), finite16<BF16>(o.y), finite16<BF16>(o.z), finite16<BF16>(o.w));
                            const int b = k0 + key - fresh;
                            if ((o.x ^ v.x) | (o.y ^ v.y) | (o.z ^ v.z) | (o.w ^ v.w)) {
                                atomicOr(&s_odd[b >> 5], 1u << (b & 31));
                                __threadfence_block();  // the other row tile, which finds the zeros, finds the bit
                            }
                        }
                        *at_x = v;
                    }
                    fence_proxy_async();
                }
                const float ms = (m == -INFINITY ? 0.0f : m) - kAtLift<BF16>;
                const uint64_t scales = pack2(scale, scale), shift = pack2(-ms, -ms);
                uint64_t sums[2] = {0, 0};
                {
                    float *x = s;
                    // For 16-bit outputs one pair of eight goes to a polynomial: the exponential unit (16 a cycle) would take
                    // 1024 cycles for the 64 x 256 weights of a step, the warps' other instructions fewer issue slots.  An
                    // fp32 output's terms leave no slots for that.
                    if (plain) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint64_t y = fma2(pack2(x[2 * e], x[2 * e + 1]), scales, shift);
                            if (!F32 && (e & 7) < 1) {
                                exp2_poly<BF16 ? 4 : 5>(y, x[2 * e], x[2 * e + 1]);
                            } else {
                                unpack2(y, x[2 * e], x[2 * e + 1]);
                                x[2 * e] = ex2(x[2 * e]);
                                x[2 * e + 1] = ex2(x[2 * e + 1]);
                            }
                            sums[e & 1] = add2(sums[e & 1], pack2(x[2 * e], x[2 * e + 1]));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = (see >> e) & 1u ? ex2(fmaf(x[e], scale, -ms)) : 0.0f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) sums[e & 1] = add2(sums[e & 1], pack2(x[2 * e], x[2 * e + 1]));
                    }
                    // All terms but the last are cut off, not rounded: what is left is exact, and takes one operation a pair.
#pragma unroll
                    for (int t = 0; t < T::TERMS; ++t) {
                        uint32_t u[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            if (t + 1 == T::TERMS) {
                                u[e] = pack16<BF16>(x[2 * e], x[2 * e + 1]);
                                continue;
                            }
                            constexpr uint32_t kKeep = BF16 ? 0xffff0000u : 0xffffe000u;
                            const float a = __uint_as_float(__float_as_uint(x[2 * e]) & kKeep), b = __uint_as_float(__float_as_uint(x[2 * e + 1]) & kKeep);
                            u[e] = BF16 ? __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632) : pack16<BF16>(a, b);
                            unpack2(fma2(pack2(a, b), pack2(-1.0f, -1.0f), pack2(x[2 * e], x[2 * e + 1])), x[2 * e], x[2 * e + 1]);
                        }
                        tmem_st16(region + hf * (16 * T::TERMS) + t * 16, u);
                    }
                }
                {
                    float a, b;
                    unpack2(add2(sums[0], sums[1]), a, b);
                    l += a + b;
                }
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                mbar_arrive_lane0(pfull + 8 * buf, lane);
            }
            // the segment's partial result
            const int unit = at.seq < 0 ? at.kvh * P.tcm_pre + at.mt
                                        : nkv * P.tcm_pre + (at.seq * nkv + at.kvh) * P.tcm_own + at.mt;
            const long long to = P.tc_row0 + ((long long)unit + c) * T::ROWS + w * 128;
            if (tid == 0 && t0 == 0) P.tc_cta_of[unit].x = c;
            if (tid == 0 && t0 + n + kTcEmpty == at.tiles) P.tc_cta_of[unit].y = c;
            if (mine) {
                um_spin(odone + 8 * w, oph, fail);
                oph ^= 1u;
                tmem_fence_after();
            }
            // the halves' sums meet (the maxima are the same); nobody reads the other turn's any more
            s_top[turn][w][hf][row] = l;
            rows_sync(w, warp & 3);
            if (hf == 0 && r < M) P.ml[to + row] = make_float2(m, l + s_top[turn][w][1][row]);
            turn ^= 1;
            tile_sync(w);                   // all its warps have looked at the last tiles' values
            const int late = keys - fresh;  // new slots there are
            const unsigned long long there = late >= 64 ? ~0ull : late <= 0 ? 0ull : (1ull << late) - 1;
            // ... and those of them in this partial's tiles: another's infinite value times the weight zero of a partial that
            // has seen nothing would be NaN.  The 64 new slots lie in two tiles at the most.
            const int j0 = fresh / N - t0, first_new = N - fresh % N;  // the first one's tile of the segment, its new slots
            const unsigned long long low = first_new >= 64 ? ~0ull : (1ull << first_new) - 1;
            const auto of_mine = [&](int j) { return j >= 0 && j < n && (!two || (j & 1) == w); };
            const unsigned long long here = (of_mine(j0) ? low : 0ull) | (of_mine(j0 + 1) ? ~low : 0ull);
            const unsigned long long odd = (s_odd[0] | (unsigned long long)s_odd[1] << 32) & bits & there & here;
            // A thread has a row's dims, a store wants a row's dims in neighbouring lanes: 32 rows x CW dims at a time turn in the
            // shared memory of this row tile's query vectors, whose products are done.  Wide pieces of a row fill whole lines of
            // the partial results (with 16 dims at a time, and 8 loads of query vectors under way, the call above took 50 us).
            constexpr int CW = D == 64 ? 16 : 32, CL = CW / 4;  // lanes of a row
            uint8_t *swap = base + w * T::Q_BYTES + (warp & 7) * (CW * 128);
#pragma unroll 1
            for (int d = hf * (D / 2); d < (hf + 1) * (D / 2); d += CW) {
                float o[CW];
#pragma unroll
                for (int h = 0; h < CW; h += 16) {
                    float v[16];
                    if (mine) {
                        tmem_ld16(tmem + lanes + T::O_COL + w * D + d + h, v);
                        tmem_wait_ld16(v);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[h + e] = mine ? v[e] : 0.0f;
                }
                for (unsigned long long q = odd; q; q &= q - 1) {
                    const uint16_t *v = P.own.v + (long long)at.seq * P.own.seq_stride + at.kvh * P.own.head_stride +
                                        ((long long)fresh + __ffsll(q) - 1) * P.own.slot_stride + d;
#pragma unroll
                    for (int e = 0; e < CW; ++e) {
                        const float x = from16<BF16>(v[e]);
                        if (!isfinite(x)) o[e] += x;
                    }
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < CL; ++e)
                    *reinterpret_cast<float4 *>(swap + lane * (CW * 4) + ((e ^ turn_at(lane, CL)) << 4)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < CL; ++e) {
                    const int rr = e * (32 / CL) + lane / CL, ch = lane % CL;
                    const float4 v = *reinterpret_cast<const float4 *>(swap + rr * (CW * 4) + ((ch ^ turn_at(rr, CL)) << 4));
                    if (r - lane + rr < M) *reinterpret_cast<float4 *>(P.part + (to + (row & ~31) + rr) * D + d + ch * 4) = v;
                }
            }
            tile_sync(w);  // before new query vectors replace what another warp still turns
            ring.skip(2 * n % T::SLOTS);
            if ((2 * n / T::SLOTS) & 1) ring.ph ^= 1u;
            tmem_fence_before();
        }
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if (tid == 0 && *fail) {
        report_error(P.err, kErrBarrierTimeout);
        const long long t0 = clock64();  // copies that are under way land before the shared memory is given back
        while (clock64() - t0 < 4000000LL) {
        }
    }
    __syncthreads();
    if (warp == kIssuer) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace pgb
