// Entry points of the attention half of a decode layer: query/key norms with rotation and cache store, attention
// behind a shared prefix, cache eviction.  Declared in include/peregrine_b200.h.
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <mutex>
#include <vector>

#include "../../include/peregrine_b200.h"
#include "ctx.h"
#include "kernels_attn_tc.cuh"
#include "kernels_evict.cuh"
#include "kernels_norm_rope.cuh"
#include "kv_overlap.h"

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
    for (const long long s : {a->seq_stride, a->head_stride, a->slot_stride})  // the copy engine's strides end at 2^40 bytes
        if (s < 0 || s >= 1ll << 39 || (s & 7)) return refuse("%s: cache strides must be multiples of 8", what);
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

// What a call of the attention and the question for its scratch have in common.
int attn_ok(int S, int H, const KvArgs &own, int prefix_len, int rows_per_seq, const char *what) {
    if (!rows_ok(S, H, own, rows_per_seq, what)) return 0;
    if (rows_per_seq > 64) return refuse("%s: %d rows of a sequence are more than 64", what, rows_per_seq);
    if (H % own.n_kv) return refuse("%s: %d heads are no multiple of %d", what, H, own.n_kv);
    if (prefix_len < 0) return refuse("%s: negative prefix", what);
    if ((long long)S * H > 0x3fffffff || (own.acc && ((long long)own.cap / 32 + 1) * own.n_seq * own.n_kv > 0x3fffffff))
        return refuse("%s: too many rows and heads", what);
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

// Dynamic shared-memory opt-in, once per kernel and device (cudaFuncSetAttribute takes a microsecond of every call otherwise).
struct OptIn {
    const void *fn;
    int device, bytes;
};
std::mutex g_opt_mu;
std::vector<OptIn> g_opt;

template <typename K>
int opt_in(K kernel, int bytes) {
    const void *fn = reinterpret_cast<const void *>(kernel);
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return refuse("shared-memory opt-in: no current device");
    std::lock_guard<std::mutex> lk(g_opt_mu);
    for (OptIn &e : g_opt)
        if (e.fn == fn && e.device == device) {
            if (e.bytes >= bytes) return 1;
            const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (r == cudaSuccess) e.bytes = bytes;
            return r == cudaSuccess ? 1 : refuse("shared-memory opt-in: %s", cudaGetErrorString(r));
        }
    const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (r != cudaSuccess) return refuse("shared-memory opt-in: %s", cudaGetErrorString(r));
    g_opt.push_back({fn, device, bytes});
    return 1;
}

// A launch that may start while the one before it in the stream still runs: every kernel here sets itself up, waits on the
// device for what came before (the one launch that need not says so), and only then lets the next one start.  `early` false:
// an ordinary launch.  A grid that fills the device is placed unevenly while the one before still holds some SMs: six
// sequences' eviction took 59 us early and 52 in order, a split of two long sequences 83 and 70; a call of one sequence 9.5
// early and 12.3 in order.
template <typename... K, typename... A>
int launch_early(void (*kernel)(K...), unsigned grid, int block, int smem, cudaStream_t stream, const char *what, int cluster, bool early,
                 A... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = early;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, K(args)...);
    return launched(what);
}

struct NormRopeLaunch {
    NormRopeArgs &P;
    int S, sms;
    cudaStream_t stream;
    template <int D, bool BF16>
    int operator()() const {
        // a warp gets a stretch of items: as long ones as leave none without
        const int warps = kNrPerSm * kNrWarps * sms, steps = ((P.H + 2 * P.kv.n_kv) * D + 255) / 256;
        const long long all = (long long)S * steps;
        P.rows = S;
        P.steps = steps;
        const long long per = (all + warps - 1) / warps;
        P.per = (int)(per > kNrSteps ? kNrSteps : per);
        P.parts = (steps + P.per - 1) / P.per;
        if ((long long)S * P.parts > 0x7fffffffll) return refuse("pipe_qk_norm_rope: too many rows and heads");
        const long long need = ((long long)S * P.parts + kNrWarps - 1) / kNrWarps, most = (long long)kNrPerSm * sms;
        auto kernel = P.R & 7 ? norm_rope_kernel<D, BF16, false> : norm_rope_kernel<D, BF16, true>;
        if (!opt_in(kernel, kNrSmem)) return 0;
        return launch_early(kernel, (unsigned)(need < most ? need : most), kNrWarps * 32, kNrSmem, stream,
                            "qk_norm_rope launch", 1, true, P);
    }
};

// Problems with more row vectors than this go to the tensor-memory kernel, whose tiles have 128 rows (both sides: kAtMany).
constexpr int kTcRows = kAtMany;

// Row tile of the split kernel.
int row_tile(int rows, int H, int n_kv) { return rows * (H / n_kv) <= 8 ? 8 : 16; }
// Its CTAs: as many as are resident at once.
int attn_ctas(int D, int rt, int sms) {
    if (D == 64) return sms * (rt == 8 ? SplitShape<64, 8>::PER_SM : SplitShape<64, 16>::PER_SM);
    if (D == 128) return sms * (rt == 8 ? SplitShape<128, 8>::PER_SM : SplitShape<128, 16>::PER_SM);
    return sms * (rt == 8 ? SplitShape<256, 8>::PER_SM : SplitShape<256, 16>::PER_SM);
}

// Shapes and the scratch's layout from the description of a call; bytes needed, or 0 for numbers past the kernels' range.
size_t attn_plan(AttnArgs *P, const KvArgs &own, int S, int H, int prefix_len, int rows, int sms, char *work) {
    const long long m_own = (long long)rows * (H / own.n_kv), m_pre = (long long)S * (H / own.n_kv);
    P->G = H / own.n_kv;
    const int rt = row_tile(rows, H, own.n_kv);
    P->tc_pre = prefix_len && m_pre > kTcRows;
    P->tc_own = m_own > kTcRows;
    const long long mt_own = P->tc_own ? 0 : (m_own + rt - 1) / rt, mt_pre = prefix_len && !P->tc_pre ? (m_pre + rt - 1) / rt : 0;
    const long long units = own.n_kv * (mt_pre + own.n_seq * mt_own);
    P->tc_rows = own.D == 256 ? 128 : 256;
    P->tc_ctas = sms;
    P->tc2_pre = own.D < 256 && m_pre <= 128;
    P->tc2_own = own.D < 256 && m_own <= 128;
    const long long tcm_pre = P->tc_pre ? (m_pre + P->tc_rows - 1) / P->tc_rows : 0, tcm_own = P->tc_own ? (m_own + P->tc_rows - 1) / P->tc_rows : 0;
    const long long tc_units = own.n_kv * (tcm_pre + own.n_seq * tcm_own), tiles = (long long)own.cap / 64 + 16;
    // units and the tiles of one sequence are counted in 32 bits
    if (units > 0x3fffffff || tc_units > 0x3fffffff || m_pre > 0x3fffffff || tiles * own.n_kv * (mt_own > tcm_own ? mt_own : tcm_own) > 0x3fffffff)
        return 0;
    P->mt_own = (int)mt_own;
    P->mt_pre = (int)mt_pre;
    P->tcm_pre = (int)tcm_pre;
    P->tcm_own = (int)tcm_own;
    P->ctas = units ? attn_ctas(own.D, rt, sms) : 0;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *p = work ? work + at : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t split_rows = ((size_t)units + P->ctas) * rt, tc_rows = tc_units ? ((size_t)tc_units + P->tc_ctas) * P->tc_rows : 0;
    P->tc_row0 = (long long)split_rows;
    P->part = reinterpret_cast<float *>(take((split_rows + tc_rows) * own.D * 4));
    P->ml = reinterpret_cast<float2 *>(take((split_rows + tc_rows) * 8));
    P->cta_of = reinterpret_cast<int2 *>(take((size_t)units * 8));
    P->tc_cta_of = reinterpret_cast<int2 *>(take((size_t)tc_units * 8));
    P->scores = own.acc ? reinterpret_cast<float *>(take((size_t)own.n_seq * own.n_kv * m_own * (((size_t)own.cap + 3) / 4) * 16)) : nullptr;
    P->stats = own.acc ? reinterpret_cast<float2 *>(take((size_t)S * H * 8)) : nullptr;
    return at;
}

// Copies of [64 keys][64 dims] boxes of a cache, swizzled by 128 bytes; slots from `slots` on come as zeros.
int kv_map(CUtensorMap *m, const void *p, const KvArgs &kv, int slots, int dtype) {
    typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const EncodeFn enc = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &st) != cudaSuccess || st != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return (EncodeFn)fn;
    }();
    if (!enc) return 0;
    // a stride of a dimension with one entry is never used, but has to be a valid one
    const long long head = kv.n_kv > 1 ? kv.head_stride : kv.slot_stride, seq = kv.n_seq > 1 ? kv.seq_stride : kv.slot_stride;
    const cuuint64_t dims[4] = {(cuuint64_t)kv.D, (cuuint64_t)slots, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_seq};
    const cuuint64_t strides[3] = {(cuuint64_t)kv.slot_stride * 2, (cuuint64_t)head * 2, (cuuint64_t)seq * 2};
    const cuuint32_t box[4] = {64, kAtKeys, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(p), dims, strides,
               box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct AttnLaunch {
    const AttnArgs &P;
    const CUtensorMap *maps;  // of the prefix's and the own keys and values
    cudaStream_t stream;
    template <int D, bool BF16, bool F32, int RT>
    int run() const {
        constexpr int kSmem = SplitShape<D, RT>::SMEM;
        auto split = attn_split_kernel<D, BF16, F32, RT>;
        if (P.ctas && !opt_in(split, kSmem)) return 0;
        if (P.tc_pre || P.tc_own) {
            using T = TcShape<D, BF16, F32>;
            static_assert(T::ROWS == (D == 256 ? 128 : 256), "as planned");
            auto tc = attn_tc_kernel<D, BF16, F32>;
            if (!opt_in(tc, T::SMEM)) return 0;
            if (!launch_early(tc, P.tc_ctas, T::THREADS, T::SMEM, stream, "attention tensor launch", 1, true, P, maps[0], maps[1], maps[2], maps[3]))
                return 0;
        }
        if (P.ctas) {  // (behind the tensor-memory kernel it fills the SMs that this leaves, and ends after it)
            const long long tiles = (long long)P.own.n_kv * ((long long)P.own.n_seq * P.mt_own * (P.own.cap / kAtKeys + 1) +
                                                             (long long)P.mt_pre * (P.prefix_len / kAtKeys + 1));  // at the most
            const bool early = P.tc_pre || tiles <= 2 * P.ctas;
            if (!launch_early(split, P.ctas, kAtThreads, kSmem, stream, "attention launch", 1, early, P, maps[0], maps[1], maps[2], maps[3]))
                return 0;
        }
        // waits on the device for the end of the launches before
        const int vectors = P.S * P.H, groups = P.own.n_seq * P.own.n_kv;
        const bool few = vectors < 16 * P.tc_ctas, many = P.tc_own;
        const int row_ctas = few ? vectors : (vectors + 3) / 4, chunks = P.own.acc && !many ? (P.own.cap + kAtChunk - 1) / kAtChunk : 0;
        if (!launch_early(few ? attn_join_kernel<D, BF16, 4> : attn_join_kernel<D, BF16, 1>, (unsigned)(row_ctas + chunks * groups), kAtCombine,
                          0, stream, "attention join launch", 1, true, P, RT, row_ctas, chunks))
            return 0;
        if (!P.own.acc || !many) return 1;
        const int parts = (P.own.cap + 31) / 32;
        return launch_early(attn_acc_kernel, (unsigned)(parts * groups), 256, 0, stream, "attention weights launch", 1, true, P, parts);
    }
    template <int D, bool BF16>
    int operator()() const {
        if (row_tile(P.rows, P.H, P.own.n_kv) == 8) return P.out_f32 ? run<D, BF16, true, 8>() : run<D, BF16, false, 8>();
        return P.out_f32 ? run<D, BF16, true, 16>() : run<D, BF16, false, 16>();
    }
};

}  // namespace

void pgb::forget_opt_ins() {
    std::lock_guard<std::mutex> lk(g_opt_mu);
    g_opt.clear();
}

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
    if (row_stride > (1ll << 60) / S) return refuse("%s: row stride %lld is too large for %d rows", what, row_stride, S);
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(q_out), x0 = reinterpret_cast<uintptr_t>(qkv_dev),
                    x_bytes = ((uintptr_t)(S - 1) * row_stride + ((uintptr_t)H + 2ull * kv->n_kv) * kv->D) * 4;  // to the last row's last value
    if (q0 < x0 + x_bytes && x0 < q0 + (uintptr_t)S * H * kv->D * 2) return refuse("%s: q_out overlaps the rows", what);
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
    P.log2_theta = R ? std::log2((double)theta) : 0.0;
    P.R = R;
    P.style = style;
    if (!ctx_of(device, &c)) return refuse("%s: device %d is not initialised", what, device);
    P.err = c.err;
    DeviceGuard g(c.device);
    if (!g.ok()) return refuse("%s: device %d cannot be selected", what, device);
    return by_type(kv->D, kv->dtype, NormRopeLaunch{P, S, c.sms, c.stream});
}

PGB_EXPORT size_t coli_cuda_pipe_attention_workspace(int device, int S, int H, const ColiCudaKv *own, int prefix_len,
                                                     int rows_per_seq) {
    const char *what = "pipe_attention_workspace";
    CtxRef c;
    KvArgs kv;
    if (!kv_args(&kv, own, what) || !attn_ok(S, H, kv, prefix_len, rows_per_seq, what)) return 0;
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
    if (!kv_args(&P.own, own, what) || !attn_ok(S, H, P.own, prefix_len, rows_per_seq, what)) return 0;
    if (!out_dev || !q_dev || !base_dev || !work_dev) return refuse("%s: null pointer", what);
    if (!aligned(out_dev, 16) || !aligned(q_dev, 16) || !aligned(base_dev, 4) || !aligned(mask_dev, 8) || !aligned(work_dev, 256))
        return refuse("%s: misaligned pointer", what);
    if (out_f32 != 0 && out_f32 != 1) return refuse("%s: out_f32 is not 0 or 1", what);
    if (prefix_len) {
        if (!kv_args(&P.pre, prefix, what)) return 0;
        if (prefix->n_seq != 1 || prefix->n_kv != own->n_kv || prefix->D != own->D || prefix->dtype != own->dtype)
            return refuse("%s: the prefix is not one sequence of the cache's heads and type", what);
        if (prefix_len > prefix->cap) return refuse("%s: prefix of %d slots in a cache of %d", what, prefix_len, prefix->cap);
    }
    if (!std::isfinite(scale * 1.4426950408889634f)) return refuse("%s: scale is not finite in units of log2(e)", what);
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
    P.err = c.err;
    DeviceGuard g(c.device);
    if (!g.ok()) return refuse("%s: device %d cannot be selected", what, device);
    CUtensorMap maps[4] = {};
    const int type = own->dtype;
    if ((prefix_len && !(kv_map(&maps[0], P.pre.k, P.pre, prefix_len, type) && kv_map(&maps[1], P.pre.v, P.pre, prefix_len, type))) ||
        !(kv_map(&maps[2], P.own.k, P.own, P.own.cap, type) && kv_map(&maps[3], P.own.v, P.own, P.own.cap, type)))
        return refuse("%s: the cache cannot be described to the copy engine", what);
    if (!prefix_len) {  // not used
        maps[0] = maps[2];
        maps[1] = maps[3];
    }
    return by_type(own->D, own->dtype, AttnLaunch{P, maps, c.stream});
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
    if (!same) {
        const auto all = [](const KvArgs &a, Rows *r) {
            for (const void *p : {a.k, a.v})
                *r++ = {addr(p), (Wide)a.seq_stride * 2, (Wide)a.head_stride * 2, (Wide)a.slot_stride * 2, a.n_seq, a.n_kv, a.cap, a.D * 2};
            for (const void *p : {(const void *)a.pos, (const void *)a.acc}) *r++ = {addr(p), 0, 0, 0, 1, 1, 1, (Wide)a.n_seq * a.n_kv * a.cap * 4};
        };
        Rows to[4], from[4];
        all(P.dst, to);
        all(P.src, from);
        for (const Rows &d : to)
            for (const Rows &f : from)
                if (rows_meet(d, f)) return refuse("%s: source and target share some of their memory", what);
    }
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
    if (src->cap > kEvCluster * kEvPartMost) {
        if (!launch_early(evict_select_kernel, (unsigned)groups, kEvThreads, 0, c.stream, "kv_evict select launch", 1, false, P)) return 0;
    } else {
        const int parts = src->cap <= kEvAlone ? 1 : kEvCluster, most = (((src->cap + parts - 1) / parts) + 7) & ~7, smem = most * 6;
        auto kernel = parts == 1 ? evict_select_cluster_kernel<1> : evict_select_cluster_kernel<kEvCluster>;
        if (!opt_in(kernel, smem)) return 0;
        if (!launch_early(kernel, (unsigned)(groups * parts), kEvPartThreads, smem, c.stream, "kv_evict select launch", parts, groups * parts <= c.sms, P, most))
            return 0;
    }
    const int per_cta = 4 * 256 / (src->D / 8);
    const long long most = ((long long)keep + per_cta - 1) / per_cta, want = (16ll * c.sms + groups - 1) / groups;
    P.chunks = (int)(most < want ? most : want);
    auto move = src->D == 64 ? evict_move_kernel<64> : src->D == 128 ? evict_move_kernel<128> : evict_move_kernel<256>;
    return launch_early(move, (unsigned)(groups * P.chunks), 256, 0, c.stream, "kv_evict move launch", 1, true, P);
}
