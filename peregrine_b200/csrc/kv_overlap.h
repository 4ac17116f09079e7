// Whether the memory of two strided caches meets (host only).
#pragma once
#include <algorithm>
#include <cstdint>

namespace pgb {

typedef __int128 Wide;  // strides up to 2^40 bytes times counts up to 2^31
inline Wide addr(const void *p) { return (Wide) reinterpret_cast<uintptr_t>(p); }

// Memory that a cache's rows take: `width` bytes each, strides in bytes.
struct Rows {
    Wide at, seq, head, slot;
    int n_seq, n_kv, cap;
    Wide width;
    Wide block() const { return (cap - 1) * slot + width; }      // bytes of one (sequence, head), gaps and all
    Wide blocks() const { return (n_kv - 1) * head + block(); }  // of a sequence
};
// Which of the spans [y + j * step, + each), j < n, meet [x, x + bytes): first to last, none where last < first.
struct Meeting {
    int first, last;
    Meeting(Wide x, Wide bytes, Wide y, Wide step, Wide each, int n) {
        const Wide before = x - y - each, behind = x + bytes - y;  // j * step lies between the two
        if (n == 1 || step == 0) {
            first = 0, last = before < 0 && behind > 0 ? n - 1 : -1;
            return;
        }
        first = before < 0 ? 0 : (int)std::min<Wide>(before / step + 1, n);
        last = behind <= 0 ? -1 : (int)std::min<Wide>((behind - 1) / step, n - 1);
    }
    bool any() const { return first <= last; }
};
// Whether two caches' rows share a byte.  Rows of one may lie between the other's (layers or heads side by side, slots in turn), so
// where the spans of two heads meet, their rows decide.  Past a million such looks (tens of milliseconds) the caches count as shared.
inline bool rows_meet(const Rows &a, const Rows &b) {
    long long looks = 1 << 20;
    if (!Meeting(a.at, (a.n_seq - 1) * a.seq + a.blocks(), b.at, 0, (b.n_seq - 1) * b.seq + b.blocks(), 1).any()) return false;
    for (int s = 0; s < a.n_seq; ++s) {
        const Wide x = a.at + s * a.seq;
        const Meeting of(x, a.blocks(), b.at, b.seq, b.blocks(), b.n_seq);
        if (--looks < 0) return true;
        for (int t = of.first; t <= of.last; ++t)
            for (int h = 0; h < a.n_kv; ++h) {
                const Wide p = x + h * a.head;
                const Meeting heads(p, a.block(), b.at + t * b.seq, b.head, b.block(), b.n_kv);
                if (--looks < 0) return true;
                for (int g = heads.first; g <= heads.last; ++g) {
                    const Wide q = b.at + t * b.seq + g * b.head;
                    if (--looks < 0) return true;
                    if (a.cap > 1 && b.cap > 1 && a.slot == b.slot) {
                        // rows i and j: only p - q + (i - j) * slot counts, so the first of either against all of the other
                        if (Meeting(p, a.width, q, b.slot, b.width, b.cap).any() || Meeting(q, b.width, p, a.slot, a.width, a.cap).any())
                            return true;
                        continue;
                    }
                    const bool less = a.cap < b.cap;
                    const Rows &few = less ? a : b, &many = less ? b : a;
                    if ((looks -= few.cap) < 0) return true;
                    for (int i = 0; i < few.cap; ++i)
                        if (Meeting((less ? p : q) + i * few.slot, few.width, less ? q : p, many.slot, many.width, many.cap).any()) return true;
                }
            }
    }
    return false;
}

}  // namespace pgb
