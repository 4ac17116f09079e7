// Eviction: the best `keep` slots of every (sequence, kv head) by rank, moved to the front.
//
// A slot's rank is one 32-bit key: the accumulated weight as an order-preserving integer, all ones for protected
// slots, zero for NaN; ties go to the lower slot.  A radix select of 8 bits a pass finds the smallest kept key and
// how many of its ties are kept; one ordered sweep then pairs the m-th free place below `keep` with the m-th kept
// slot behind it.  Only those rows move, so nothing is read after it was overwritten when the cache is its own target.
#pragma once
#include <limits.h>

#include "kernels_norm_rope.cuh"

namespace pgb {

struct EvictArgs {
    KvArgs dst, src;
    const int *len;
    int *new_len, *index;
    int keep, sinks, recent;
    int chunks;  // CTAs that share the moves of one (sequence, kv head)
};

constexpr int kEvThreads = 1024;

// Order-preserving key of one slot: larger is kept first.
__device__ __forceinline__ uint32_t evict_key(float acc, int pos, int last, int sinks, int recent) {
    if (pos < sinks || (long long)pos > (long long)last - recent) return 0xFFFFFFFFu;
    if (acc != acc) return 0u;
    const uint32_t u = __float_as_uint(acc + 0.0f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive sum of one value per thread over the CTA in thread order; `total` gets the sum.
__device__ __forceinline__ int block_scan(int v, int *s_warp, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int before = 0, all = 0;
    const int w = s_warp[lane];  // kEvThreads / 32 == 32 warps
    int y = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    all = __shfl_sync(0xffffffffu, y, 31);
    before = __shfl_sync(0xffffffffu, y - w, warp);
    total = all;
    return before + x - v;
}

// One CTA for caches whose keys do not fit into a cluster's shared memory: every sweep forms them anew.
__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const EvictArgs P) {
    __shared__ int s_warp[32], s_hist[256], s_digit, s_above, s_last;
    const int seq = blockIdx.x / P.src.n_kv;
    griddep_wait();
    griddep_launch_dependents();
    int len = P.len[seq];
    if (len < 0) return;
    len = min(len, P.src.cap);
    const int count = min(len, P.keep), tid = threadIdx.x;
    const long long at = (long long)blockIdx.x * P.src.cap;
    const float *acc = P.src.acc + at;
    const int *pos = P.src.pos + at;
    int *index = P.index + (long long)blockIdx.x * P.keep;
    for (int i = count + tid; i < P.keep; i += kEvThreads) index[i] = -1;
    if (len <= P.keep) {
        for (int i = tid; i < count; i += kEvThreads) index[i] = i;
        return;
    }
    if (tid == 0) s_last = INT_MIN;
    __syncthreads();
    int last = INT_MIN;
    for (int i = tid; i < len; i += kEvThreads) last = max(last, pos[i]);
    last = __reduce_max_sync(0xffffffffu, last);
    if ((tid & 31) == 0) atomicMax(&s_last, last);
    __syncthreads();
    last = s_last;
    // radix select: `prefix` = the digits of the count-th largest key found so far, `want` = its rank among equals
    uint32_t prefix = 0;
    int want = count;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < len; i += kEvThreads) {
            const uint32_t key = evict_key(acc[i], pos[i], last, P.sinks, P.recent);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        int total;
        const int mine = tid < 256 ? s_hist[255 - tid] : 0;
        const int above = block_scan(mine, s_warp, total);  // keys of a larger digit
        if (tid < 256 && above < want && above + mine >= want) {
            s_digit = 255 - tid;
            s_above = above;
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        want -= s_above;
        __syncthreads();
    }
    // `want` of the slots with this very key are kept, the lowest ones.  Slots from `keep` on that are kept are
    // listed in index[0..] in order; places below `keep` then take them, from the top down, so that an entry of the
    // list (never above the place that takes it) is read before its own place is written.
    int ties = 0, moved = 0;
    const int rounds = (len + kEvThreads - 1) / kEvThreads;
    int holes_all = 0;
    for (int r = 0; r < rounds; ++r) {
        const int i = r * kEvThreads + tid;
        const uint32_t key = i < len ? evict_key(acc[i], pos[i], last, P.sinks, P.recent) : 0u;
        const bool tie = i < len && key == prefix;
        int n, m;
        const int t = ties + block_scan(tie, s_warp, n);
        ties += n;
        const bool kept = i < len && (key > prefix || (tie && t < want));
        const bool far = kept && i >= P.keep;
        const int f = moved + block_scan(far, s_warp, m);
        if (far) index[f] = i;
        moved += m;
        holes_all += __syncthreads_count(!kept && i < P.keep && i < len);
    }
    int holes = holes_all, tie_end = 0;  // tie_end: ties below the current round, found by counting down
    const int low = (P.keep + kEvThreads - 1) / kEvThreads;
    for (int r = 0; r < low; ++r) {  // ties below `keep`
        const int i = r * kEvThreads + tid;
        tie_end += __syncthreads_count(i < P.keep && evict_key(acc[i], pos[i], last, P.sinks, P.recent) == prefix);
    }
    for (int r = low - 1; r >= 0; --r) {
        const int i = r * kEvThreads + tid;
        const bool in = i < P.keep;
        const uint32_t key = in ? evict_key(acc[i], pos[i], last, P.sinks, P.recent) : 0u;
        const bool tie = in && key == prefix;
        int n, m;
        const int t = block_scan(tie, s_warp, n);
        tie_end -= n;
        const bool kept = in && (key > prefix || (tie && tie_end + t < want));
        const bool hole = in && !kept;
        const int rank = block_scan(hole, s_warp, m);
        holes -= m;
        int from = i;
        if (hole) from = index[holes + rank];
        __syncthreads();
        if (in) index[i] = from;
        __syncthreads();
    }
}

// The same on a cluster of C CTAs (kEvCluster, or 1 for short caches) per (sequence, kv head): every CTA keeps the keys of its
// part of the slots in shared memory, histograms and counts are read across the cluster.  Measured for 48 times
// up to 40000 slots: one CTA each 108 us, clusters of eight 33 (the whole call 52; with clusters of four 65); what is left are the
// exchanges (about 1 us each, seven of them) and the sweeps between them.
constexpr int kEvCluster = 8, kEvPartThreads = 512, kEvPartMost = 32768;  // slots of a CTA at the most
// Slots up to which one CTA is a cluster.  us of a call with one CTA / with clusters, 1, 8 and 32 sequences of 8 heads: 1000 slots
// 9.7 / 15.5, 13.8 / 20.1 and 40.9 / 76.3; 1500 slots 13.2 / 14.4, 24.2 / 22.8 and 53.1 / 76.8; 4000 slots 16.2 / 16.7, 52.9 / 45.1, 133.8 / 151.7.
constexpr int kEvAlone = 1024;

template <int C>
__device__ __forceinline__ void cluster_sync() {
    if (C == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}
template <int C>
__device__ __forceinline__ int cluster_ld(const int *p, int rank) {  // *p of CTA `rank` of the cluster
    if (C == 1) return *p;
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return (int)v;
}
template <int C>
__device__ __forceinline__ int cluster_ld16(const uint16_t *p, int rank) {
    if (C == 1) return *p;
    uint32_t a;
    uint16_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
    return v;
}

template <int C>
__global__ void __launch_bounds__(kEvPartThreads) evict_select_cluster_kernel(const EvictArgs P, int part_most) {
    constexpr int W = kEvPartThreads / 32;
    static_assert(kEvPartThreads >= 256, "a thread per digit");
    extern __shared__ __align__(16) uint32_t ev_key[];
    uint16_t *surv = reinterpret_cast<uint16_t *>(ev_key + part_most);  // the part's kept slots behind `keep`, in order
    __shared__ int s_hist[2][256], s_last, s_ties, s_far, s_holes, s_digit, s_above, s_warp[3][W];
    const int rank = C == 1 ? 0 : blockIdx.x % C, g = blockIdx.x / C, seq = g / P.src.n_kv;
    griddep_wait();
    griddep_launch_dependents();
    int len = P.len[seq];
    if (len < 0) return;
    len = min(len, P.src.cap);
    const int count = min(len, P.keep), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int *index = P.index + (long long)g * P.keep;
    for (int i = count + rank * kEvPartThreads + tid; i < P.keep; i += C * kEvPartThreads) index[i] = -1;
    if (len <= P.keep) {
        for (int i = rank * kEvPartThreads + tid; i < count; i += C * kEvPartThreads) index[i] = i;
        return;
    }
    const int part = (len + C - 1) / C, lo = min(rank * part, len), n = min(part, len - lo);
    const float *acc = P.src.acc + (long long)g * P.src.cap + lo;
    const int *pos = P.src.pos + (long long)g * P.src.cap + lo;
    if (tid == 0) s_last = INT_MIN, s_ties = s_far = s_holes = 0;
    if (tid < 256) s_hist[0][tid] = s_hist[1][tid] = 0;
    __syncthreads();
    int last = INT_MIN;
#pragma unroll 8
    for (int i = tid; i < n; i += kEvPartThreads) {
        last = max(last, pos[i]);
        ev_key[i] = __float_as_uint(acc[i]);
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) atomicMax(&s_last, last);
    cluster_sync<C>();
#pragma unroll
    for (int r = 0; r < C; ++r) last = max(r ? last : INT_MIN, cluster_ld<C>(&s_last, r));
#pragma unroll 8
    for (int i = tid; i < n; i += kEvPartThreads) ev_key[i] = evict_key(__uint_as_float(ev_key[i]), pos[i], last, P.sinks, P.recent);
    __syncthreads();
    // radix select: `prefix` = the digits of the count-th largest key found so far, `want` = its rank among equals
    uint32_t prefix = 0;
    int want = count;
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        int *hist = s_hist[pass & 1];
        for (int i0 = warp * 32; i0 < n; i0 += 4 * kEvPartThreads) {
            int digit[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * kEvPartThreads + lane;
                const uint32_t key = i < n ? ev_key[i] : 0u;
                const bool in = i < n && (pass == 0 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
                digit[u] = in ? (int)((key >> shift) & 255) : -1;
            }
            if (pass == 0) {  // weights share their leading digits: one addition for a warp's equal ones
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t same = __match_any_sync(0xffffffffu, digit[u]);
                    if (digit[u] >= 0 && (same & ((1u << lane) - 1)) == 0) atomicAdd(&hist[digit[u]], __popc(same));
                }
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (digit[u] >= 0) atomicAdd(&hist[digit[u]], 1);
            }
        }
        cluster_sync<C>();
        int mine = 0;
        if (tid < 256) {
#pragma unroll
            for (int r = 0; r < C; ++r) mine += cluster_ld<C>(&hist[255 - tid], r);
            s_hist[(pass + 1) & 1][tid] = 0;  // read by all before this barrier
        }
        int x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s_warp[0][warp] = x;
        __syncthreads();
        int above = x - mine;  // keys of a larger digit
#pragma unroll
        for (int w = 0; w < W; ++w) above += w < warp ? s_warp[0][w] : 0;
        if (tid < 256 && above < want && above + mine >= want) {
            s_digit = 255 - tid;
            s_above = above;
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        want -= s_above;
    }
    // Warps own runs of the part: `want` of the slots with this very key are kept, the lowest ones.
    const int run = (n + W * 32 - 1) / (W * 32) * 32, a0 = min(warp * run, n), a1 = min(a0 + run, n);
    int ties = 0;
#pragma unroll 4
    for (int i = a0 + lane; i < a0 + run; i += 32) ties += i < a1 && ev_key[i] == prefix;
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) {
        s_warp[0][warp] = ties;
        atomicAdd(&s_ties, ties);
    }
    cluster_sync<C>();
    int before = 0;
    for (int r = 0; r < rank; ++r) before += cluster_ld<C>(&s_ties, r);
    for (int w = 0; w < warp; ++w) before += s_warp[0][w];
    // One word of kept flags for every 32 slots, in the place of their first key.
    const uint32_t below = (1u << lane) - 1;
#pragma unroll 4
    for (int i0 = a0, t = before; i0 < a1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < a1 ? ev_key[i] : 0u;
        const uint32_t tb = __ballot_sync(0xffffffffu, i < a1 && key == prefix);
        const uint32_t kept = __ballot_sync(0xffffffffu, i < a1 && (key > prefix || (key == prefix && t + __popc(tb & below) < want)));
        t += __popc(tb);
        if (lane == 0) ev_key[i0] = kept;
    }
    __syncwarp();
    // of a word: the slots before `keep`, kept ones behind it, free ones before it
    auto low_of = [&](int i0) { return P.keep - lo - i0 >= 32 ? 0xffffffffu : P.keep - lo - i0 <= 0 ? 0u : (1u << (P.keep - lo - i0)) - 1; };
    auto in_of = [&](int i0) { return a1 - i0 >= 32 ? 0xffffffffu : (1u << (a1 - i0)) - 1; };
    int far = 0, holes = 0;
    for (int i0 = a0 + 32 * lane; i0 < a1; i0 += 1024) {
        const uint32_t kept = ev_key[i0], low = low_of(i0);
        far += __popc(kept & ~low);
        holes += __popc(in_of(i0) & ~kept & low);
    }
    far = __reduce_add_sync(0xffffffffu, far);
    holes = __reduce_add_sync(0xffffffffu, holes);
    if (lane == 0) {
        s_warp[1][warp] = far;
        s_warp[2][warp] = holes;
        atomicAdd(&s_far, far);
        atomicAdd(&s_holes, holes);
    }
    __syncthreads();
    int f = 0, h = 0;
    for (int w = 0; w < warp; ++w) {
        f += s_warp[1][w];
        h += s_warp[2][w];
    }
#pragma unroll 4
    for (int i0 = a0; i0 < a1; i0 += 32) {
        const uint32_t fk = ev_key[i0] & ~low_of(i0);
        if ((fk >> lane) & 1u) surv[f + __popc(fk & below)] = (uint16_t)(i0 + lane);
        f += __popc(fk);
    }
    cluster_sync<C>();
    int fars[C];  // kept slots behind `keep` in the parts before the r-th
    {
        int sum = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) {
            fars[r] = sum;
            sum += cluster_ld<C>(&s_far, r);
            if (r < rank) h += cluster_ld<C>(&s_holes, r);
        }
    }
#pragma unroll 2
    for (int i0 = a0; i0 < a1 && lo + i0 < P.keep; i0 += 32) {
        const uint32_t kept = ev_key[i0], low = low_of(i0), hk = in_of(i0) & ~kept & low;
        if ((hk >> lane) & 1u) {
            const int m = h + __popc(hk & below);
            int r = 0, first = 0;
#pragma unroll
            for (int q = 1; q < C; ++q)
                if (fars[q] <= m) r = q, first = fars[q];
            index[lo + i0 + lane] = r * part + cluster_ld16<C>(&surv[m - first], r);
        } else if ((kept & low) >> lane & 1u) {
            index[lo + i0 + lane] = lo + i0 + lane;
        }
        h += __popc(hk);
    }
    cluster_sync<C>();  // nobody leaves while its shared memory is read
}

// Moves the selected rows: 16 bytes a lane, D / 8 lanes for a row of k and of v, four rows under way at a time.  Bound by HBM:
// 48 x 2048 rows of 2 x 256 bytes in 17.3 us, 5.6 TB/s read and written.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs P) {
    constexpr int LPR = D / 8, ROWS = 256 / LPR, U = 4;
    const int g = blockIdx.x / P.chunks, chunk = blockIdx.x % P.chunks, seq = g / P.src.n_kv, kvh = g % P.src.n_kv;
    griddep_wait();
    griddep_launch_dependents();
    const int len = P.len[seq];
    const int count = min(min(len, P.src.cap), P.keep);  // (negative for padding, which keeps its length)
    if (kvh == 0 && chunk == 0 && threadIdx.x == 0) P.new_len[seq] = len < 0 ? len : count;
    if (len < 0) return;
    const bool in_place = P.dst.k == P.src.k;
    const int sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const long long sb = (long long)seq * P.src.seq_stride + kvh * P.src.head_stride + l * 8;
    const long long db = (long long)seq * P.dst.seq_stride + kvh * P.dst.head_stride + l * 8;
    for (int i0 = chunk * (ROWS * U) + sub; i0 < count; i0 += P.chunks * (ROWS * U)) {
        int from[U];
        uint4 a[U], b[U];
        int p[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * ROWS;
            from[u] = i < count ? P.index[(long long)g * P.keep + i] : -1;
            if (in_place && from[u] == i) from[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (from[u] >= 0) {
                a[u] = *reinterpret_cast<const uint4 *>(P.src.k + sb + from[u] * P.src.slot_stride);
                b[u] = *reinterpret_cast<const uint4 *>(P.src.v + sb + from[u] * P.src.slot_stride);
                if (l == 0) {
                    p[u] = P.src.pos[(long long)g * P.src.cap + from[u]];
                    w[u] = P.src.acc[(long long)g * P.src.cap + from[u]];
                }
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (from[u] >= 0) {
                const int i = i0 + u * ROWS;
                *reinterpret_cast<uint4 *>(P.dst.k + db + i * P.dst.slot_stride) = a[u];
                *reinterpret_cast<uint4 *>(P.dst.v + db + i * P.dst.slot_stride) = b[u];
                if (l == 0) {
                    P.dst.pos[(long long)g * P.dst.cap + i] = p[u];
                    P.dst.acc[(long long)g * P.dst.cap + i] = w[u];
                }
            }
    }
}

}  // namespace pgb
