// Entry points of the attention half of a decode layer: query/key norms with rotation and cache store, attention
// behind a shared prefix, cache eviction.  Declared in include/peregrine_b200.h.
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/peregrine_b200.h"
#include "ctx.h"
#include "kernels_attn.cuh"
#include "kernels_evict.cuh"
#include "kernels_norm_rope.cuh"

using namespace pgb;

#define PGB_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

__attribute__((format(printf, 1, 2))) int refuse(const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::fputs("[CUDA] ", stderr);
    std::vfprintf(stderr, fmt, ap);
    std::fputc('\n', stderr);
    va_end(ap);
    return 0;
}

int launched(const char *what) {
    count_launches(1);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 1 : refuse("%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The cache as the kernels take it; 0 and a message when the description does not hold together.
int kv_args(KvArgs *a, const ColiCudaKv *kv, const char *what) {
    if (!kv || !kv->k || !kv->v) return refuse("%s: no cache", what);
    if (kv->n_seq < 1 || kv->n_kv < 1 || kv->cap < 1) return refuse("%s: empty cache shape", what);
    if (kv->D != 64 && kv->D != 128 && kv->D != 256) return refuse("%s: head width %d is not 64, 128 or 256", what, kv->D);
    if (kv->dtype != 1 && kv->dtype != 2) return refuse("%s: cache type %d is not 1 (bf16) or 2 (f16)", what, kv->dtype);
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return refuse("%s: cache not aligned to 16 bytes", what);
    if (!aligned(kv->pos, 4) || !aligned(kv->acc, 4)) return refuse("%s: pos or acc not aligned", what);
    *a = KvArgs{static_cast<uint16_t *>(kv->k), static_cast<uint16_t *>(kv->v), kv->pos, kv->acc, kv->n_seq, kv->n_kv,
                kv->cap, kv->D, kv->seq_stride, kv->head_stride, kv->slot_stride};
    if (!kv->seq_stride && !kv->head_stride && !kv->slot_stride) {
        a->slot_stride = kv->D;
        a->head_stride = (long long)kv->cap * kv->D;
        a->seq_stride = (long long)kv->n_kv * a->head_stride;
    }
    const long long limit = 1ll << 44;  // offsets stay far from 64-bit overflow
    for (const long long s : {a->seq_stride, a->head_stride, a->slot_stride})
        if (s < 0 || s > limit || (s & 7)) return refuse("%s: cache strides must be multiples of 8", what);
    if (a->slot_stride < kv->D || (kv->n_kv > 1 && a->head_stride < kv->D) || (kv->n_seq > 1 && a->seq_stride < kv->D))
        return refuse("%s: cache strides overlap", what);
    return 1;
}

int rows_ok(int S, int H, const KvArgs &kv, int rows_per_seq, const char *what) {
    if (S < 1 || H < 1 || rows_per_seq < 1) return refuse("%s: empty call", what);
    if (H > 65536 || kv.n_kv > 65536) return refuse("%s: too many heads", what);
    if ((long long)kv.n_seq * rows_per_seq != S) return refuse("%s: %d rows are not %d sequences of %d", what, S, kv.n_seq, rows_per_seq);
    return 1;
}

template <typename F>
int by_type(int D, int dtype, F &&f) {  // f.template operator()<D, BF16>()
    if (dtype == 1) {
        if (D == 64) return f.template operator()<64, true>();
        if (D == 128) return f.template operator()<128, true>();
        return f.template operator()<256, true>();
    }
    if (D == 64) return f.template operator()<64, false>();
    if (D == 128) return f.template operator()<128, false>();
    return f.template operator()<256, false>();
}

struct NormRopeLaunch {
    const NormRopeArgs &P;
    int S, sms;
    cudaStream_t stream;
    template <int D, bool BF16>
    int operator()() const {
        // a CTA takes all heads of a row once the rows alone fill the device a few times over
        const int per_cta = kNrWarps * (256 / D), groups = (P.H + 2 * P.kv.n_kv + per_cta - 1) / per_cta;
        const int split = S >= 8 * sms ? 1 : groups;
        norm_rope_kernel<D, BF16><<<dim3(S, split < 65535 ? split : 65535), kNrWarps * 32, 0, stream>>>(P);
        return launched("qk_norm_rope launch");
    }
};

int row_tile(long long m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

// CTAs of the split kernel: as many as are resident at once (shared memory of a CTA: 73, 113 or 193 kB).
int attn_ctas(int D, int sms) { return sms * (D == 64 ? 3 : D == 128 ? 2 : 1); }

// Shapes and the scratch's layout from the description of a call; bytes needed, or 0 for numbers past the kernels' range.
size_t attn_plan(AttnArgs *P, const KvArgs &own, int S, int H, int prefix_len, int rows, int sms, char *work) {
    const long long m_own = (long long)rows * (H / own.n_kv), m_pre = (long long)S * (H / own.n_kv);
    P->G = H / own.n_kv;
    P->rt_own = row_tile(m_own);
    P->rt_pre = row_tile(m_pre);
    P->rt_max = prefix_len ? (P->rt_pre > P->rt_own ? P->rt_pre : P->rt_own) : P->rt_own;
    const long long mt_own = (m_own + P->rt_own - 1) / P->rt_own, mt_pre = prefix_len ? (m_pre + P->rt_pre - 1) / P->rt_pre : 0;
    const long long units = own.n_kv * (mt_pre + own.n_seq * mt_own);
    if (units > 0x3fffffff || m_pre > 0x3fffffff) return 0;
    P->mt_own = (int)mt_own;
    P->mt_pre = (int)mt_pre;
    P->ctas = attn_ctas(own.D, sms);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = work ? work + at : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t rows_all = (size_t)(units + P->ctas) * P->rt_max;
    P->part = reinterpret_cast<float *>(take(rows_all * own.D * 4));
    P->ml = reinterpret_cast<float2 *>(take(rows_all * 8));
    P->offs = reinterpret_cast<int *>(take(((size_t)own.n_seq + 1) * 4));
    P->scores = own.acc ? reinterpret_cast<float *>(take((size_t)own.n_seq * own.n_kv * m_own * own.cap * 4)) : nullptr;
    return at;
}

template <typename K>
int opt_in(K kernel, int bytes) {  // per device and cheap: set on every launch that needs it
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == cudaSuccess ? 1 : refuse("shared-memory opt-in: %s", cudaGetErrorString(e));
}

struct AttnLaunch {
    const AttnArgs &P;
    cudaStream_t stream;
    template <int D, bool BF16>
    int operator()() const {
        auto split = P.out_f32 ? attn_split_kernel<D, BF16, true> : attn_split_kernel<D, BF16, false>;
        if (!opt_in(split, kAtSmem<D>)) return 0;
        split<<<dim3(P.ctas), kAtThreads, kAtSmem<D>, stream>>>(P);
        if (!launched("attention launch")) return 0;
        // the joining launch starts early and waits on the device for the first one's end
        const int chunks = P.own.acc ? (P.own.cap + 2 * kAtCombine - 1) / (2 * kAtCombine) : 0;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3((unsigned)((long long)P.S * P.H + (long long)chunks * P.own.n_seq * P.own.n_kv));
        cfg.blockDim = dim3(kAtCombine);
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, attn_join_kernel<D, BF16>, P, chunks);
        return launched("attention join launch");
    }
};

}  // namespace

PGB_EXPORT int coli_cuda_pipe_qk_norm_rope(int device, void *q_out, const float *qkv_dev, long long row_stride, int S,
                                           int H, const ColiCudaKv *kv, const float *q_w, const float *k_w, float eps,
                                           const int *pos_dev, const int *base_dev, int rows_per_seq, float theta,
                                           int R, int style) {
    const char *what = "pipe_qk_norm_rope";
    CtxRef c;
    NormRopeArgs P{};
    if (!kv_args(&P.kv, kv, what) || !rows_ok(S, H, P.kv, rows_per_seq, what)) return 0;
    if (!q_out || !qkv_dev || !pos_dev || !base_dev) return refuse("%s: null pointer", what);
    if (!aligned(q_out, 16) || !aligned(qkv_dev, 16) || (row_stride & 3)) return refuse("%s: rows not aligned to 16 bytes", what);
    if (!aligned(q_w, 4) || !aligned(k_w, 4) || !aligned(pos_dev, 4) || !aligned(base_dev, 4)) return refuse("%s: misaligned pointer", what);
    if (row_stride < ((long long)H + 2ll * kv->n_kv) * kv->D || row_stride > (1ll << 40)) return refuse("%s: row stride %lld is too small or large", what, row_stride);
    if (R < 0 || R > kv->D || (R & 1)) return refuse("%s: rotary width %d is not an even number up to %d", what, R, kv->D);
    if (style != 0 && style != 1) return refuse("%s: style %d is not 0 or 1", what, style);
    if (R && !(theta > 0.0f && theta < 3e38f)) return refuse("%s: theta must be positive", what);
    if (!(eps >= 0.0f)) return refuse("%s: eps must not be negative", what);
    P.q_out = static_cast<uint16_t *>(q_out);
    P.qkv = qkv_dev;
    P.row_stride = row_stride;
    P.H = H;
    P.q_w = q_w;
    P.k_w = k_w;
    P.eps = eps;
    P.pos = pos_dev;
    P.base = base_dev;
    P.rows_per_seq = rows_per_seq;
    P.theta = theta;
    P.R = R;
    P.style = style;
    if (!ctx_of(device, &c)) return refuse("%s: device %d is not initialised", what, device);
    DeviceGuard g(c.device);
    if (!g.ok()) return refuse("%s: device %d cannot be selected", what, device);
    return by_type(kv->D, kv->dtype, NormRopeLaunch{P, S, c.sms, c.stream});
}

PGB_EXPORT size_t coli_cuda_pipe_attention_workspace(int device, int S, int H, const ColiCudaKv *own, int prefix_len,
                                                     int rows_per_seq) {
    const char *what = "pipe_attention_workspace";
    CtxRef c;
    KvArgs kv;
    if (!kv_args(&kv, own, what) || !rows_ok(S, H, kv, rows_per_seq, what)) return 0;
    if (prefix_len < 0 || H % kv.n_kv || rows_per_seq > 64) return (size_t)refuse("%s: shape", what);
    if (!ctx_of(device, &c)) return (size_t)refuse("%s: device %d is not initialised", what, device);
    AttnArgs P{};
    const size_t need = attn_plan(&P, kv, S, H, prefix_len, rows_per_seq, c.sms, nullptr);
    return need ? need : (size_t)refuse("%s: too many rows and heads", what);
}

PGB_EXPORT int coli_cuda_pipe_attention(int device, void *out_dev, int out_f32, const void *q_dev, int S, int H,
                                        const ColiCudaKv *prefix, int prefix_len, const ColiCudaKv *own,
                                        const int *base_dev, int rows_per_seq, const uint64_t *mask_dev, float scale,
                                        void *work_dev, size_t work_bytes) {
    const char *what = "pipe_attention";
    CtxRef c;
    AttnArgs P{};
    if (!kv_args(&P.own, own, what) || !rows_ok(S, H, P.own, rows_per_seq, what)) return 0;
    if (rows_per_seq > 64) return refuse("%s: %d rows of a sequence are more than 64", what, rows_per_seq);
    if (H % own->n_kv) return refuse("%s: %d heads are no multiple of %d", what, H, own->n_kv);
    if ((long long)S * H + (own->acc ? (long long)(own->cap / 256 + 1) * own->n_seq * own->n_kv : 0) > 0x7fffffffll)
        return refuse("%s: too many rows and heads", what);
    if (!out_dev || !q_dev || !base_dev || !work_dev) return refuse("%s: null pointer", what);
    if (!aligned(out_dev, 16) || !aligned(q_dev, 16) || !aligned(base_dev, 4) || !aligned(mask_dev, 8) || !aligned(work_dev, 256))
        return refuse("%s: misaligned pointer", what);
    if (out_f32 != 0 && out_f32 != 1) return refuse("%s: out_f32 is not 0 or 1", what);
    if (prefix_len < 0) return refuse("%s: negative prefix", what);
    if (prefix_len) {
        if (!kv_args(&P.pre, prefix, what)) return 0;
        if (prefix->n_seq != 1 || prefix->n_kv != own->n_kv || prefix->D != own->D || prefix->dtype != own->dtype)
            return refuse("%s: the prefix is not one sequence of the cache's heads and type", what);
        if (prefix_len > prefix->cap) return refuse("%s: prefix of %d slots in a cache of %d", what, prefix_len, prefix->cap);
    }
    if (!(scale == scale) || scale - scale != 0.0f) return refuse("%s: scale is not finite", what);
    P.out = out_dev;
    P.out_f32 = out_f32;
    P.q = static_cast<const uint16_t *>(q_dev);
    P.S = S;
    P.H = H;
    P.prefix_len = prefix_len;
    P.base = base_dev;
    P.rows = rows_per_seq;
    P.mask = reinterpret_cast<const unsigned long long *>(mask_dev);
    P.scale2 = scale * 1.4426950408889634f;
    if (!ctx_of(device, &c)) return refuse("%s: device %d is not initialised", what, device);
    const size_t need = attn_plan(&P, P.own, S, H, prefix_len, rows_per_seq, c.sms, static_cast<char *>(work_dev));
    if (!need) return refuse("%s: too many rows and heads", what);
    if (work_bytes < need) return refuse("%s: %zu bytes of workspace, %zu are needed", what, work_bytes, need);
    DeviceGuard g(c.device);
    if (!g.ok()) return refuse("%s: device %d cannot be selected", what, device);
    return by_type(own->D, own->dtype, AttnLaunch{P, c.stream});
}

PGB_EXPORT int coli_cuda_pipe_kv_evict(int device, const ColiCudaKv *dst, const ColiCudaKv *src, const int *len_dev,
                                       int *new_len_dev, int *index_dev, int keep, int sinks, int recent) {
    const char *what = "pipe_kv_evict";
    CtxRef c;
    EvictArgs P{};
    if (!kv_args(&P.src, src, what) || !kv_args(&P.dst, dst, what)) return 0;
    if (dst->n_seq != src->n_seq || dst->n_kv != src->n_kv || dst->D != src->D || dst->dtype != src->dtype)
        return refuse("%s: source and target differ in shape or type", what);
    if (!src->pos || !src->acc || !dst->pos || !dst->acc) return refuse("%s: pos and acc are needed in both caches", what);
    if (!len_dev || !new_len_dev || !index_dev) return refuse("%s: null pointer", what);
    if (!aligned(len_dev, 4) || !aligned(new_len_dev, 4) || !aligned(index_dev, 4)) return refuse("%s: misaligned pointer", what);
    if (keep < 1 || keep > dst->cap) return refuse("%s: %d slots cannot be kept in a cache of %d", what, keep, dst->cap);
    if (sinks < 0 || recent < 0) return refuse("%s: negative sinks or recent", what);
    const bool same_k = dst->k == src->k, same = same_k && dst->v == src->v && dst->pos == src->pos && dst->acc == src->acc &&
                        P.dst.cap == P.src.cap && P.dst.seq_stride == P.src.seq_stride &&
                        P.dst.head_stride == P.src.head_stride && P.dst.slot_stride == P.src.slot_stride;
    if (!same && (same_k || dst->v == src->v || dst->pos == src->pos || dst->acc == src->acc))
        return refuse("%s: source and target share some of their memory", what);
    const long long groups = (long long)src->n_seq * src->n_kv;
    if (groups > 1 << 20) return refuse("%s: too many sequences and heads", what);
    P.len = len_dev;
    P.new_len = new_len_dev;
    P.index = index_dev;
    P.keep = keep;
    P.sinks = sinks;
    P.recent = recent;
    if (!ctx_of(device, &c)) return refuse("%s: device %d is not initialised", what, device);
    DeviceGuard g(c.device);
    if (!g.ok()) return refuse("%s: device %d cannot be selected", what, device);
    evict_select_kernel<<<dim3((unsigned)groups), kEvThreads, 0, c.stream>>>(P);
    if (!launched("kv_evict select launch")) return 0;
    const int per_cta = 256 / (src->D / 8);
    const long long most = ((long long)keep + per_cta - 1) / per_cta, want = (16ll * c.sms + groups - 1) / groups;
    P.chunks = (int)(most < want ? most : want);
    const dim3 grid((unsigned)(groups * P.chunks));
    if (src->D == 64)
        evict_move_kernel<64><<<grid, 256, 0, c.stream>>>(P);
    else if (src->D == 128)
        evict_move_kernel<128><<<grid, 256, 0, c.stream>>>(P);
    else
        evict_move_kernel<256><<<grid, 256, 0, c.stream>>>(P);
    return launched("kv_evict move launch");
}
