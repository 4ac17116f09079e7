"""The attention operators against their formulas in 64 bits: sizes, masks and memory layouts where they can go wrong."""
import ctypes as C

import numpy as np
import pytest
import torch

from peregrine_b200 import attention as at, cuda
from tests import attention_ref as ref
from tests.attention_ref import HALF, TYPES, f64, i32

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------- norm, rotation, store
def run_norm(seed, n, r, H, Kv, D, R, style, T, cap, base, pos, q_norm=True, k_norm=True, pad=0, slot_major=False,
             theta=1e4, eps=1e-6):
    rng = np.random.default_rng(seed)
    S = n * r
    x = (1.5 * rng.standard_normal((S, (H + 2 * Kv) * D + pad))).astype(np.float32)
    wq, wk = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    k, v = (ref.cache(rng, n, Kv, cap, D, T, slot_major) for _ in range(2))
    k0, v0 = f64(k), f64(v)
    slots = torch.full((n, Kv, cap), -7, dtype=torch.int32, device="cuda")
    acc = torch.full((n, Kv, cap), 3.0, device="cuda")
    q = torch.full((S, H, D), 9.0, dtype=TYPES[T], device="cuda")
    dev = [torch.from_numpy(a).cuda() for a in (x, wq, wk)]
    b, p = i32(base), i32(pos)
    torch.cuda.synchronize()
    at.qk_norm_rope(0, q.data_ptr(), dev[0].data_ptr(), S, H, ref.view(k, v, T, slots, acc), b.data_ptr(), p.data_ptr(),
                    theta, rotary=R, style=style, q_weight=dev[1].data_ptr() if q_norm else 0,
                    k_weight=dev[2].data_ptr() if k_norm else 0, eps=eps, rows_per_seq=r, row_stride=x.shape[1])
    ref.done()
    xx = x[:, :(H + 2 * Kv) * D].astype(np.float64).reshape(S, H + 2 * Kv, D)
    ang = np.asarray(pos, np.float64)[:, None] * np.float64(np.float32(theta)) ** (-2.0 * np.arange(R // 2) / max(R, 1))
    cs, sn = np.cos(ang)[:, None, :], np.sin(ang)[:, None, :]

    def turned(t, w):
        if w is not None:
            t = t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * w
        a, bb = (t[..., 0:R:2], t[..., 1:R:2]) if style == 0 else (t[..., :R // 2], t[..., R // 2:R])
        size = np.concatenate([np.abs(a) + np.abs(bb)] * 2 + [np.abs(t[..., R:])], -1)
        return np.concatenate([a * cs - bb * sn, bb * cs + a * sn, t[..., R:]], -1), size

    def near(got, want, size):
        # fp32: the norm's sum of D squares and its root (D/2 + 4 half steps), cosine and rotation a few more; one rounding
        tol = np.abs(want) * HALF[T] + size * (D / 2 + 16) * 2.0 ** -24 * (1 + HALF[T]) + (2.0 ** -25 if T == "f16" else 0)
        assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())

    wantq, sq = turned(xx[:, :H], wq if q_norm else None)
    wantk, sk = turned(xx[:, H:H + Kv], wk if k_norm else None)
    gq, gk, gv, gs, ga = f64(q), f64(k), f64(v), slots.cpu().numpy(), acc.cpu().numpy()
    for s in range(S):
        bb, i = divmod(s, r)
        if base[bb] < 0:
            assert np.all(gq[s] == 9.0)
            continue
        near(gq[s], wantq[s], sq[s])
        t = base[bb] + i
        if t < cap:
            near(gk[bb, :, t], wantk[s], sk[s])
            vr = f64(torch.from_numpy(x[s, (H + Kv) * D:(H + 2 * Kv) * D].reshape(Kv, D)).to(TYPES[T]))
            assert np.array_equal(gv[bb, :, t], vr)
            assert np.all(gs[bb, :, t] == pos[s]) and np.all(ga[bb, :, t] == 0.0)
            k0[bb, :, t], v0[bb, :, t] = gk[bb, :, t], gv[bb, :, t]
            gs[bb, :, t], ga[bb, :, t] = -7, 3.0
    # nothing else of the cache was touched
    assert np.array_equal(gk, k0) and np.array_equal(gv, v0) and np.all(gs == -7) and np.all(ga == 3.0)


@pytest.mark.parametrize("T", ["bf16", "f16"])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("D, R", [(64, 64), (64, 62), (64, 24), (128, 128), (128, 0), (128, 2), (128, 126), (256, 256),
                                  (256, 64), (256, 254)])
def test_norm_rope_widths(dev, D, R, style, T):
    run_norm(D + R, n=3, r=2, H=5, Kv=1, D=D, R=R, style=style, T=T, cap=9, base=[0, 4, 7],
             pos=[0, 1, 4, 5, 1000000, 2147483647], pad=4)


@pytest.mark.parametrize("n, r, H, Kv, slot_major", [(1, 1, 1, 1, False), (1, 1, 48, 8, True), (5, 3, 7, 7, True),
                                                     (1, 1300, 4, 2, False), (2, 650, 3, 1, True)])
def test_norm_rope_rows(dev, n, r, H, Kv, slot_major):
    run_norm(n + r, n, r, H, Kv, 128, 128, 0, "bf16", r + 3, [3] * n, np.arange(n * r) + 3, slot_major=slot_major)


def test_norm_rope_padding_and_full_caches(dev):
    run_norm(1, 4, 3, 4, 2, 64, 64, 1, "bf16", 8, [-1, 6, 8, 2147483646], np.arange(12) - 5)
    run_norm(2, 4, 3, 4, 2, 64, 64, 0, "f16", 8, [0, -5, 5, 7], np.arange(12), q_norm=False)
    run_norm(3, 1, 2, 4, 2, 64, 32, 0, "f16", 8, [0], [3, 3], k_norm=False, theta=500000.0, eps=0.1)


# --------------------------------------------------------------------------------------- attention
def run_attention(seed, n, r, H, Kv, D, T, cap, base, Tp=0, out_f32=True, acc=False, mask=None, slot_major=False, q_std=2.0,
                  scale=None, prepare=None, check=True):
    rng = np.random.default_rng(seed)
    S = n * r
    q = torch.from_numpy((q_std * rng.standard_normal((S, H, D))).astype(np.float32)).to(TYPES[T]).cuda()
    k, v = (ref.cache(rng, n, Kv, cap, D, T, slot_major) for _ in range(2))
    pk = pv = None
    if Tp:
        pk, pv = (ref.cache(rng, 1, Kv, Tp + 5, D, T, slot_major) for _ in range(2))
    # slots behind the used ones hold what memory held before: they must not count
    for b in range(n):
        e = max(0, base[b] + r) if base[b] >= 0 else 0
        k[b, :, e:], v[b, :, e:] = float("nan"), float("inf")
    if Tp:
        pk[:, :, Tp:], pv[:, :, Tp:] = float("inf"), float("nan")
    if prepare is not None:
        prepare(q, k, v, pk, pv)
    a = torch.from_numpy(rng.random((n, Kv, cap), dtype=np.float32)).cuda()
    a0 = f64(a)
    out = torch.full((S, H, D), 7.0, dtype=torch.float32 if out_f32 else TYPES[T], device="cuda")
    bdev = i32(base)
    m = None if mask is None else torch.from_numpy(np.asarray(mask, np.uint64).view(np.int64)).cuda()
    own = ref.view(k, v, T, acc=a if acc else None)
    pre = ref.view(pk, pv, T) if Tp else None
    scale = D ** -0.5 if scale is None else scale
    need = at.attention_workspace(0, S, H, own, Tp, r)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaN everywhere: nothing of it is counted on
    torch.cuda.synchronize()

    def call():
        at.attention(0, out.data_ptr(), q.data_ptr(), S, H, own, bdev.data_ptr(), scale, work.data_ptr(), need, rows_per_seq=r,
                     prefix=pre, prefix_len=Tp, mask=0 if m is None else m.data_ptr(), out_f32=out_f32)
        ref.done()

    call()
    first, first_a = out.clone(), a.clone()
    assert cuda.last_device_error(0) == 0
    if check:
        want, wacc, gam, mag = ref.attend(f64(q), f64(k), f64(v), base, r, scale, f64(pk)[0, :, :Tp] if Tp else None,
                                          f64(pv)[0, :, :Tp] if Tp else None, mask)
        tol = ref.bound(gam, mag, Tp + cap + 64, want, T, out_f32)
        got = f64(first)
        for b in range(n):
            rows = slice(b * r, (b + 1) * r)
            if base[b] < 0:
                assert np.all(got[rows] == 7.0)
            else:
                off = np.abs(got[rows] - want[rows]) / tol[rows]
                assert np.all(off <= 1.0), float(np.nanmax(off))
        if acc:
            # a weight is off by what the output's are, the sum over rows and heads of the group by a rounding each
            t = wacc * (2 * gam.max() + 2.0 ** -20 + (Tp + cap + 64) * 2.0 ** -24) + (a0 + wacc) * (r * H // Kv + 2) * 2.0 ** -24 + 1e-30
            off = np.abs(f64(first_a) - a0 - wacc) / t
            assert np.all(off <= 1.0), float(np.nanmax(off))
        else:
            assert np.array_equal(f64(first_a), a0)
    # the same bits again, whatever the scratch held
    a.copy_(torch.from_numpy(a0.astype(np.float32)))
    torch.cuda.synchronize()
    call()
    assert torch.equal(out, first) or bool((torch.isnan(out) == torch.isnan(first)).all())
    assert torch.equal(a.nan_to_num(5.0), first_a.nan_to_num(5.0))
    return f64(first), f64(first_a) - a0


@pytest.mark.parametrize("T", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("out_f32", [True, False])
def test_attention_types(dev, D, T, out_f32):
    run_attention(D, 3, 1, 8, 2, D, T, 200, [0, 63, 199], Tp=70, out_f32=out_f32, acc=True)
    run_attention(D + 1, 2, 4, 6, 2, D, T, 150, [60, 146], Tp=129, out_f32=out_f32, acc=True, slot_major=True)


@pytest.mark.parametrize("own", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 191, 257, 1000])
def test_attention_own_lengths(dev, own):
    run_attention(own, 2, 1, 4, 2, 64, "bf16", own + 3, [own - 1, own // 2], acc=True)


@pytest.mark.parametrize("Tp", [1, 15, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_attention_prefix_lengths(dev, Tp):
    run_attention(Tp, 3, 1, 12, 2, 128, "bf16", 9, [0, 3, 8], Tp=Tp)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 33, 40])
def test_attention_groups(dev, G):
    run_attention(G, 2, 1, 2 * G, 2, 64, "f16", 90, [70, 89], Tp=40, acc=True)


@pytest.mark.parametrize("n, r", [(1, 2), (1, 7), (3, 8), (1, 16), (2, 33), (1, 63), (1, 64)])
def test_attention_rows_of_a_sequence(dev, n, r):
    run_attention(n + r, n, r, 6, 2, 128, "bf16", 130 + r, [130 - 40 * b for b in range(n)], Tp=33, acc=True)
    run_attention(n + r, n, r, 3, 3, 64, "f16", r, [0] * n, acc=True)


@pytest.mark.parametrize("n", [2, 8, 11, 16, 23, 48])
@pytest.mark.parametrize("D, out_f32, T", [(64, True, "bf16"), (128, True, "f16"), (128, False, "bf16"), (256, True, "bf16")])
def test_attention_many_rows_behind_a_prefix(dev, n, D, out_f32, T):
    """Batches whose rows fill one, two and more tiles of the shared part."""
    run_attention(n, n, 1, 16, 2, D, T, 40, [(7 * b) % 40 for b in range(n)], Tp=700, out_f32=out_f32, acc=n == 16)


@pytest.mark.parametrize("D, out_f32, T", [(64, True, "f16"), (128, False, "f16"), (128, True, "bf16"), (256, False, "bf16")])
def test_attention_more_row_vectors_than_warps(dev, D, out_f32, T):
    """Over 16 row vectors an SM: a warp joins one (two of one sequence's tiles and ten of the shared ones, and padding between)."""
    run_attention(D, 41, 1, 64, 2, D, T, 140, [-1 if b == 17 else (11 * b) % 140 for b in range(41)], Tp=1500, out_f32=out_f32)
    run_attention(D + 1, 2, 40, 32, 2, D, T, 200, [160, 3], Tp=300, out_f32=out_f32, acc=True)


def test_attention_trees_and_rows_that_see_nothing(dev):
    rng = np.random.default_rng(5)
    bits = [int(rng.integers(0, 256)) for _ in range(24)]
    run_attention(1, 3, 8, 8, 2, 64, "bf16", 300, [5, 0, 292], Tp=65, mask=bits, acc=True)
    bits[8:16] = [0] * 8  # the second sequence has no slots but its own new ones, and none of them is seen
    out, _ = run_attention(2, 3, 8, 8, 2, 128, "f16", 300, [5, 0, 292], mask=bits, acc=True)
    assert np.all(out[8:16] == 0.0)
    full = [(1 << 64) - 1] * 64
    run_attention(3, 1, 64, 2, 1, 64, "bf16", 100, [36], mask=full, acc=True)
    out, _ = run_attention(4, 2, 1, 2, 1, 64, "bf16", 4, [0, 0], mask=[0, 2], out_f32=False)  # bit 1 is no row's
    assert np.all(out == 0.0)


def test_attention_padding_sequences_and_short_caches(dev):
    run_attention(1, 5, 2, 4, 2, 64, "bf16", 50, [-1, 10, -2147483648, 48, 0], Tp=20, acc=True)
    run_attention(2, 3, 4, 4, 2, 128, "bf16", 50, [48, 49, 50], Tp=20, acc=True)  # some new slots are past the cache
    run_attention(3, 2, 1, 4, 2, 64, "bf16", 50, [-1, -1], Tp=20)
    run_attention(4, 2, 2, 4, 2, 64, "bf16", 50, [-1, -1], acc=True)
    run_attention(5, 1, 2, 4, 2, 64, "bf16", 50, [2147483646], Tp=7, acc=True)


@pytest.mark.parametrize("T", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 256])
def test_values_that_no_row_may_see(dev, T, D):
    """NaN and infinities in keys and values of new slots outside a row's mask leave the row as it is."""
    n, r, cap, base = 2, 8, 80, [60, 3]
    hidden = 5
    mask = [(1 << r) - 1 & ~(1 << hidden)] * (n * r)

    def spoil(q, k, v, pk, pv):
        for b in range(n):
            k[b, :, base[b] + hidden, ::2], k[b, :, base[b] + hidden, 1::2] = float("nan"), float("inf")
            v[b, :, base[b] + hidden, ::2], v[b, :, base[b] + hidden, 1::2] = float("-inf"), float("nan")

    clean, a0 = run_attention(3, n, r, 4, 2, D, T, cap, base, Tp=30, mask=mask, acc=True)
    out, a1 = run_attention(3, n, r, 4, 2, D, T, cap, base, Tp=30, mask=mask, acc=True, prepare=spoil, check=False)
    assert np.array_equal(out, clean) and np.array_equal(a0, a1)
    # the rows that do see such a value have it, the others do not
    seen = [m | (1 << hidden) if i % r >= 6 else m for i, m in enumerate(mask)]

    def spoil_v(q, k, v, pk, pv):
        for b in range(n):
            v[b, :, base[b] + hidden, 3] = float("inf")

    out, _ = run_attention(3, n, r, 4, 2, D, T, cap, base, Tp=30, mask=seen, prepare=spoil_v, check=False)
    for s in range(n * r):
        want_inf = s % r >= 6
        assert np.all(np.isposinf(out[s, :, 3]) == want_inf) and np.all(np.isfinite(np.delete(out[s], 3, 1)))


@pytest.mark.parametrize("T, D, heads", [("bf16", 64, 8), ("f16", 128, 24), ("bf16", 256, 12), ("f16", 64, 48)])
def test_values_that_no_row_may_see_with_many_rows(dev, T, D, heads):
    """The same where a sequence's rows fill tiles of 128 (one, two and more of them), with slots past every length spoilt."""
    n, r, cap, base, hidden = 3, 9, 210, [60, 3, 201], 5
    mask = [(1 << r) - 1 & ~(1 << hidden)] * (n * r)

    def spoil(q, k, v, pk, pv):
        for b in range(n):
            t = base[b] + hidden
            k[b, :, t, ::2], k[b, :, t, 1::2] = float("nan"), float("inf")
            v[b, :, t, ::2], v[b, :, t, 1::2] = float("-inf"), float("nan")

    clean, a0 = run_attention(3, n, r, heads, 2, D, T, cap, base, Tp=90, mask=mask, acc=True)
    out, a1 = run_attention(3, n, r, heads, 2, D, T, cap, base, Tp=90, mask=mask, acc=True, prepare=spoil, check=False)
    assert np.array_equal(out, clean) and np.array_equal(a0, a1)
    seen = [m | (1 << hidden) if i % r >= 6 else m for i, m in enumerate(mask)]

    def spoil_v(q, k, v, pk, pv):
        for b in range(n):
            v[b, :, base[b] + hidden, 3] = float("inf")

    out, _ = run_attention(3, n, r, heads, 2, D, T, cap, base, Tp=90, mask=seen, prepare=spoil_v, check=False)
    for s in range(n * r):
        want_inf = s % r >= 6
        assert np.all(np.isposinf(out[s, :, 3]) == want_inf) and np.all(np.isfinite(np.delete(out[s], 3, 1)))
    none = [0] * (n * r)
    out, _ = run_attention(4, n, r, heads, 2, D, T, r + 3, [0, 0, 0], mask=none, acc=True)
    assert np.all(out == 0.0)


def test_attention_large_scores(dev):
    """Scores of hundreds: the softmax is a single slot, and nothing overflows."""
    run_attention(1, 2, 1, 4, 2, 64, "f16", 300, [299, 50], Tp=100, q_std=40.0, scale=1.0, acc=True)
    run_attention(2, 2, 1, 4, 2, 128, "bf16", 300, [299, 50], Tp=300, q_std=40.0, scale=-1.0)


def test_attention_offsets_past_32_bits(dev):
    """Slots 2^25 elements apart: the last ones lie behind 2^32 bytes and 2^31 elements."""
    D, cap, step = 64, 70, 1 << 25
    rng = np.random.default_rng(3)
    big = torch.zeros(step * (cap - 1) + D, dtype=torch.bfloat16, device="cuda")
    k = big.as_strided((1, 1, cap, D), (0, 0, step, 1))
    k.copy_(torch.from_numpy(rng.standard_normal((1, 1, cap, D), dtype=np.float32)))
    q = torch.from_numpy(rng.standard_normal((1, 4, D), dtype=np.float32)).to(torch.bfloat16).cuda()
    out = torch.zeros((1, 4, D), device="cuda")
    own = at.KvView(k.data_ptr(), k.data_ptr(), 1, 1, cap, D, "bf16", strides=(0, 0, step))
    need = at.attention_workspace(0, 1, 4, own, cap, 1)
    work, b = torch.zeros(need, dtype=torch.uint8, device="cuda"), i32([cap - 1])
    torch.cuda.synchronize()
    at.attention(0, out.data_ptr(), q.data_ptr(), 1, 4, own, b.data_ptr(), 0.125, work.data_ptr(), need, prefix=own, prefix_len=cap)
    ref.done()
    kk = f64(k)
    want, _, gam, mag = ref.attend(f64(q), kk, kk, [cap - 1], 1, 0.125, kk[0], kk[0])
    assert np.all(np.abs(f64(out) - want) <= ref.bound(gam, mag, 2 * cap, want, "bf16", True))


def test_attention_long_splits(dev):
    """One sequence over many CTAs, and many short ones beside a long one."""
    run_attention(1, 1, 1, 4, 1, 64, "bf16", 20000, [19990], acc=True)
    run_attention(2, 1, 3, 5, 5, 128, "f16", 5000, [4997], Tp=3001)
    base = [(37 * b) % 60 for b in range(70)]
    base[33] = 3000
    run_attention(3, 70, 1, 4, 2, 64, "bf16", 3001, base, Tp=64, acc=True)


# ---------------------------------------------------------------------------------------- eviction
def run_evict(seed, n, Kv, D, cap, lens, keep, sinks, recent, T="bf16", in_place=False, slot_major=False, acc=None, pos=None,
              same_len=False, dst_cap=None):
    rng = np.random.default_rng(seed)
    k, v = (ref.cache(rng, n, Kv, cap, D, T, slot_major) for _ in range(2))
    acc = np.exp(2 * rng.standard_normal((n, Kv, cap))).astype(np.float32) if acc is None else acc
    pos = np.cumsum(rng.integers(1, 4, (n, Kv, cap)), 2).astype(np.int32) if pos is None else pos
    a, p, ln = torch.from_numpy(acc.copy()).cuda(), torch.from_numpy(pos.copy()).cuda(), i32(lens)
    k0, v0 = f64(k), f64(v)
    dc = dst_cap or keep
    if in_place:
        dk, dv, da, dp = k, v, a, p
    else:
        dk, dv = (torch.full((n, Kv, dc, D), 5.0, dtype=TYPES[T], device="cuda") for _ in range(2))
        da, dp = torch.full((n, Kv, dc), 5.0, device="cuda"), torch.full((n, Kv, dc), 5, dtype=torch.int32, device="cuda")
    index = torch.full((n, Kv, keep), 77, dtype=torch.int32, device="cuda")
    out_len = ln if same_len else torch.full((n,), 88, dtype=torch.int32, device="cuda")
    src = ref.view(k, v, T, p, a)
    dst = src if in_place else ref.view(dk, dv, T, dp, da)
    torch.cuda.synchronize()
    at.kv_evict(0, dst, src, ln.data_ptr(), out_len.data_ptr(), index.data_ptr(), keep, sinks, recent)
    ref.done()
    assert out_len.cpu().tolist() == [min(x, keep) for x in lens]
    gi, gk, gv, ga, gp = index.cpu().numpy(), f64(dk), f64(dv), da.cpu().numpy(), dp.cpu().numpy()
    for b in range(n):
        for h in range(Kv):
            if lens[b] < 0:
                assert np.all(gi[b, h] == 77)
                m = 0
            else:
                src = ref.rank_evict(pos[b, h], acc[b, h], lens[b], keep, sinks, recent)
                m = len(src)
                assert np.array_equal(gi[b, h, :m], src) and np.all(gi[b, h, m:] == -1)
                assert np.array_equal(gk[b, h, :m], k0[b, h, src]) and np.array_equal(gv[b, h, :m], v0[b, h, src])
                assert np.array_equal(ga[b, h, :m], acc[b, h, src], equal_nan=True) and np.array_equal(gp[b, h, :m], pos[b, h, src])
            rest = (k0[b, h, m:], acc[b, h, m:], pos[b, h, m:]) if in_place else (5.0, 5.0, 5)
            assert np.all(gk[b, h, m:] == rest[0]) and np.all(gp[b, h, m:] == rest[2])
            assert np.array_equal(ga[b, h, m:], np.broadcast_to(np.float32(rest[1]), ga[b, h, m:].shape), equal_nan=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D, T", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_evict(dev, D, T, in_place):
    run_evict(D, 4, 3, D, 300, [300, 120, 101, 40], 100, 4, 16, T, in_place)
    run_evict(D + 1, 2, 2, D, 3000, [2999, 1500], 1400, 0, 0, T, in_place, slot_major=True, same_len=True)


@pytest.mark.parametrize("cap, keep", [(1, 1), (2, 1), (33, 32), (1025, 1024), (1024, 1), (2050, 1025), (2049, 2048), (5000, 1023)])
def test_evict_sizes(dev, cap, keep):
    run_evict(cap + keep, 1, 2, 64, cap, [cap], keep, min(2, keep), min(3, keep), dst_cap=keep + 3)


def test_evict_ties_and_odd_weights(dev):
    rng = np.random.default_rng(0)
    n, Kv, cap = 2, 3, 2500
    few = rng.choice(np.array([0.0, -0.0, 1.0, np.inf, -np.inf, np.nan, -2.0, 1e-42], np.float32), (n, Kv, cap)).astype(np.float32)
    same = np.zeros((n, Kv, cap), np.float32)
    for acc in (few, same):
        for in_place in (False, True):
            run_evict(1, n, Kv, 64, cap, [cap, 2111], 1300, 7, 50, in_place=in_place, acc=acc)
    run_evict(2, n, Kv, 64, cap, [cap, 900], 300, 0, 1000, acc=few)  # more protected than kept: the lower slots stay
    order = np.argsort(rng.random((n, Kv, cap)), 2).astype(np.int32)  # positions in no order, as after an eviction
    run_evict(3, n, Kv, 64, cap, [cap, cap], 700, 100, 300, pos=order)
    run_evict(4, n, Kv, 64, cap, [cap, cap], 700, 2147483647, 0, acc=few)
    far = np.full((n, Kv, cap), -2147483648, np.int32)
    far[..., 5] = 2147483647
    run_evict(5, n, Kv, 64, cap, [cap, cap], 700, 0, 2147483647, pos=far)


def test_evict_lengths(dev):
    run_evict(1, 6, 1, 64, 200, [-1, 0, 1, 200, 1000, -2147483648], 50, 2, 8)
    run_evict(2, 6, 1, 64, 200, [-1, 0, 1, 200, 1000, 51], 50, 2, 8, in_place=True, same_len=True)


def test_evict_long_caches(dev):
    run_evict(1, 1, 2, 64, 60000, [60000], 4096, 4, 128)
    run_evict(2, 1, 1, 64, 130001, [130000], 65000, 4, 128, in_place=True)


def test_evict_caches_past_a_cluster(dev):
    run_evict(1, 1, 2, 64, 262145, [262145], 3000, 4, 128)
    run_evict(2, 2, 1, 64, 262144, [262144, 5000], 4000, 4, 128, in_place=True)


# --------------------------------------------------------------------------- together, and recorded
def test_calls_of_every_kernel_recorded_and_replayed(dev):
    """A graph of two attention calls (many row vectors with weights, and one row a sequence) and an eviction by a cluster,
    each with scratch of its own, replayed after the lengths, queries and weights on the device have changed: the bits of
    the same calls made directly."""
    L, rng = cuda.lib(), np.random.default_rng(7)
    n, r, H, Kv, D, cap, Tp, keep = 3, 8, 12, 2, 128, 3000, 500, 900
    k, v = (ref.cache(rng, n, Kv, cap, D, "bf16") for _ in range(2))
    pk, pv = (ref.cache(rng, 1, Kv, Tp, D, "bf16") for _ in range(2))
    dk, dv = (torch.zeros((n, Kv, keep, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pos = i32(np.broadcast_to(np.arange(cap), (n, Kv, cap)))
    acc, dacc = torch.zeros((n, Kv, cap), device="cuda"), torch.zeros((n, Kv, keep), device="cuda")
    dpos, index, new_len = i32(np.zeros((n, Kv, keep))), i32(np.zeros((n, Kv, keep))), i32([0] * n)
    q, one = (torch.zeros((m, H, D), dtype=torch.bfloat16, device="cuda") for m in (n * r, n))
    out, out1 = torch.zeros((n * r, H, D), device="cuda"), torch.zeros((n, H, D), dtype=torch.bfloat16, device="cuda")
    base, length = i32([0] * n), i32([0] * n)
    own, pre, to = ref.view(k, v, "bf16", pos, acc), ref.view(pk, pv, "bf16"), ref.view(dk, dv, "bf16", dpos, dacc)
    plain = ref.view(k, v, "bf16")
    need, need1 = at.attention_workspace(0, n * r, H, own, Tp, r), at.attention_workspace(0, n, H, plain, 0, 1)
    work, work1 = (torch.zeros(m, dtype=torch.uint8, device="cuda") for m in (need, need1))
    torch.cuda.synchronize()

    def calls():
        at.attention(0, out.data_ptr(), q.data_ptr(), n * r, H, own, base.data_ptr(), 0.1, work.data_ptr(), need, rows_per_seq=r,
                     prefix=pre, prefix_len=Tp)
        at.attention(0, out1.data_ptr(), one.data_ptr(), n, H, plain, base.data_ptr(), 0.1, work1.data_ptr(), need1,
                     out_f32=False)
        at.kv_evict(0, to, own, length.data_ptr(), new_len.data_ptr(), index.data_ptr(), keep, 4, 50)

    handle = C.c_void_p()
    assert L.coli_cuda_graph_begin(0) == 1
    calls()
    assert L.coli_cuda_graph_end(0, C.byref(handle)) == 1
    for lens in ([1000, 64, 2992], [3, 2999, 1500], [-1, 700, 901]):
        new_q, new_one = (torch.from_numpy(rng.standard_normal(t.shape, dtype=np.float32)) for t in (q, one))
        start = torch.from_numpy(rng.random((n, Kv, cap), dtype=np.float32))
        got = []
        for graph in (True, False):
            q.copy_(new_q), one.copy_(new_one), acc.copy_(start), base.copy_(i32(lens)), length.copy_(i32([x + r for x in lens]))
            for t in (out, out1, dk, dv, dacc, dpos, index, new_len):
                t.zero_()
            torch.cuda.synchronize()
            if graph:
                assert L.coli_cuda_graph_launch(handle) == 1
            else:
                calls()
            ref.done()
            got.append([t.clone() for t in (out, out1, acc, dk, dv, dacc, dpos, index, new_len)])
        for a, b in zip(*got):
            assert torch.equal(a, b)
        assert float(got[0][0].abs().sum()) > 0
    L.coli_cuda_graph_free(handle)
    assert cuda.last_device_error(0) == 0


def test_a_decode_loop_with_all_three_recorded_as_a_graph(dev):
    """Steps of norm + store, attention with weights and (at the end) an eviction, once call by call and once as a
    graph replayed on device-side lengths: the same bits, and the attention follows the lengths of the replay."""
    L = cuda.lib()
    n, H, Kv, D, cap, Tp, steps = 3, 6, 2, 64, 40, 50, 12
    rng = np.random.default_rng(0)
    pk, pv = (ref.cache(rng, 1, Kv, Tp, D, "bf16") for _ in range(2))
    rows = torch.from_numpy(rng.standard_normal((steps, n, (H + 2 * Kv) * D)).astype(np.float32)).cuda()
    results = []
    for graph in (False, True):
        k, v = (torch.zeros((n, Kv, cap, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        pos, acc = torch.zeros((n, Kv, cap), dtype=torch.int32, device="cuda"), torch.zeros((n, Kv, cap), device="cuda")
        q, out = torch.zeros((n, H, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((n, H, D), device="cuda")
        own, pre = ref.view(k, v, "bf16", pos, acc), ref.view(pk, pv, "bf16")
        base, at_pos, x = i32([0] * n), i32([0] * n), torch.zeros_like(rows[0])
        need = at.attention_workspace(0, n, H, own, Tp, 1)
        work = torch.zeros(need, dtype=torch.uint8, device="cuda")
        keep = 8
        index, new_len, length = i32(np.zeros((n, Kv, keep))), i32([0] * n), i32([steps] * n)
        torch.cuda.synchronize()

        def step():
            at.qk_norm_rope(0, q.data_ptr(), x.data_ptr(), n, H, own, base.data_ptr(), at_pos.data_ptr(), 1e4)
            at.attention(0, out.data_ptr(), q.data_ptr(), n, H, own, base.data_ptr(), 0.125, work.data_ptr(), need, prefix=pre,
                         prefix_len=Tp)

        handle = C.c_void_p()
        if graph:
            assert L.coli_cuda_graph_begin(0) == 1
            step()
            assert L.coli_cuda_graph_end(0, C.byref(handle)) == 1
        outs = []
        for t in range(steps):
            x.copy_(rows[t])
            base.fill_(t)
            at_pos.fill_(Tp + t)
            torch.cuda.synchronize()
            if graph:
                assert L.coli_cuda_graph_launch(handle) == 1
            else:
                step()
            ref.done()
            want, _, gam, mag = ref.attend(f64(q), f64(k), f64(v), [t] * n, 1, 0.125, f64(pk)[0], f64(pv)[0])
            assert np.all(np.abs(f64(out) - want) <= ref.bound(gam, mag, Tp + cap, want, "bf16", True))
            outs.append(out.clone())
        # every step gave each own slot its weights: those of a step sum to the own share of the heads
        total = f64(acc).sum((1, 2))
        assert np.all(total > 0) and np.all(total < steps * H)
        at.kv_evict(0, own, own, length.data_ptr(), new_len.data_ptr(), index.data_ptr(), keep, sinks=0, recent=3)
        ref.done()
        assert new_len.cpu().tolist() == [keep] * n
        assert all(set(range(Tp + steps - 3, Tp + steps)) <= set(row[:keep]) for row in pos.cpu().numpy().reshape(-1, cap).tolist())
        results.append(torch.stack(outs).cpu().numpy().tobytes() + k.cpu().float().numpy().tobytes() + acc.cpu().numpy().tobytes())
        if graph:
            L.coli_cuda_graph_free(handle)
    assert results[0] == results[1]
