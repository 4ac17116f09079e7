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

__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const EvictArgs P) {
    __shared__ int s_warp[32], s_hist[256], s_digit, s_above, s_last;
    const int seq = blockIdx.x / P.src.n_kv;
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

// Moves the selected rows: 16 bytes a lane, D / 8 lanes for a row of k and as many for v.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs P) {
    constexpr int LPR = D / 8;
    const int g = blockIdx.x / P.chunks, chunk = blockIdx.x % P.chunks, seq = g / P.src.n_kv, kvh = g % P.src.n_kv;
    const int len = P.len[seq];
    const int count = min(min(len, P.src.cap), P.keep);
    if (kvh == 0 && chunk == 0 && threadIdx.x == 0) P.new_len[seq] = min(len, P.keep);
    if (len < 0) return;
    const bool in_place = P.dst.k == P.src.k;
    const int sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const long long sb = (long long)seq * P.src.seq_stride + kvh * P.src.head_stride;
    const long long db = (long long)seq * P.dst.seq_stride + kvh * P.dst.head_stride;
    for (int i = chunk * (256 / LPR) + sub; i < count; i += P.chunks * (256 / LPR)) {
        const int from = P.index[(long long)g * P.keep + i];
        if (in_place && from == i) continue;
        const long long s = sb + from * P.src.slot_stride + l * 8, d = db + i * P.dst.slot_stride + l * 8;
        const uint4 a = *reinterpret_cast<const uint4 *>(P.src.k + s), b = *reinterpret_cast<const uint4 *>(P.src.v + s);
        *reinterpret_cast<uint4 *>(P.dst.k + d) = a;
        *reinterpret_cast<uint4 *>(P.dst.v + d) = b;
        if (l == 0) {
            P.dst.pos[(long long)g * P.dst.cap + i] = P.src.pos[(long long)g * P.src.cap + from];
            P.dst.acc[(long long)g * P.dst.cap + i] = P.src.acc[(long long)g * P.src.cap + from];
        }
    }
}

}  // namespace pgb
