"""Calls of the attention operators at the edges of what their declarations allow, each against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from peregrine_b200 import attention as at, cuda
from tests import attention_ref as ref
from tests.attention_ref import TYPES, f64, i32

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("cap, dst_cap, keep, lens", [
    (100, 150, 150, [200, 150, 101, 100, 99, 1, 0, -1, -5]),  # one CTA a (sequence, head)
    (100, 130, 101, [2147483647, 100, 40]),
    (3000, 3600, 3500, [4000, 3300, 3000, 2999, -1]),         # a cluster each
    (262145, 262300, 262200, [262300]),                       # longer than a cluster's shared memory
])
@pytest.mark.parametrize("same_len", [False, True])
def test_evict_lengths_past_the_source_into_a_larger_target(dev, cap, dst_cap, keep, lens, same_len):
    """A length past the source's cap counts as cap, whatever the target could take: the new length is that of the slots
    that were stored, and behind it neither the index nor the target says anything."""
    n, Kv, D = len(lens), 2, 64
    rng = np.random.default_rng(cap + keep)
    k, v = (ref.cache(rng, n, Kv, cap, D, "bf16") for _ in range(2))
    acc = torch.from_numpy(rng.random((n, Kv, cap), dtype=np.float32)).cuda()
    pos = i32(np.broadcast_to(np.arange(cap), (n, Kv, cap)))
    dk, dv = (torch.full((n, Kv, dst_cap, D), 5.0, dtype=TYPES["bf16"], device="cuda") for _ in range(2))
    dacc, dpos = torch.full((n, Kv, dst_cap), 5.0, device="cuda"), i32(np.full((n, Kv, dst_cap), 5))
    index, length = i32(np.full((n, Kv, keep), 77)), i32(lens)
    new = length if same_len else i32([88] * n)
    torch.cuda.synchronize()
    at.kv_evict(0, ref.view(dk, dv, "bf16", dpos, dacc), ref.view(k, v, "bf16", pos, acc), length.data_ptr(), new.data_ptr(),
                index.data_ptr(), keep, 2, 3)
    ref.done()
    want = [x if x < 0 else min(x, cap, keep) for x in lens]
    assert new.cpu().tolist() == want
    for b, m in enumerate(want):
        stored = max(m, 0)
        if m >= 0:
            there = torch.arange(keep, device="cuda").where(torch.arange(keep, device="cuda") < stored, -1)
            assert torch.equal(index[b], there.int().expand(Kv, keep))  # nothing was left out
        for t, f, rest in ((dk, k, 5.0), (dv, v, 5.0), (dacc, acc, 5.0), (dpos, pos, 5)):
            assert torch.equal(t[b, :, :stored], f[b, :, :stored]) and bool((t[b, :, stored:] == rest).all())


# --------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("D, T, out_f32", [(64, "bf16", True), (128, "bf16", False), (128, "f16", True), (256, "f16", False)])
def test_infinite_values_of_many_short_sequences(dev, D, T, out_f32):
    """A CTA works on several (sequence, head) pairs in a row, most with a single tile of keys: a row that sees an infinite
    value of its own sequence has an infinity there, and nothing of it is left for the next pair."""
    n, r, G, Kv, cap, hidden = 90, 9, 4, 4, 40, 5
    rng = np.random.default_rng(D)
    H, S = G * Kv, n * r
    q = torch.from_numpy(rng.standard_normal((S, H, D), dtype=np.float32)).to(TYPES[T]).cuda()
    k, v = (ref.cache(rng, n, Kv, cap, D, T) for _ in range(2))
    base = rng.integers(0, cap - r + 1, n)
    odd = np.arange(n) % 3 != 1
    for b in np.nonzero(odd)[0]:
        v[b, :, base[b] + hidden, 3] = float("inf")
        v[b, 1, base[b] + hidden, D - 2] = float("-inf")
    clean = v.clone()
    clean[~torch.isfinite(clean)] = 0.0
    out = torch.zeros((S, H, D), dtype=torch.float32 if out_f32 else TYPES[T], device="cuda")
    own, bdev = ref.view(k, v, T), i32(base)
    need = at.attention_workspace(0, S, H, own, 0, r)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(5):
        torch.cuda.synchronize()
        at.attention(0, out.data_ptr(), q.data_ptr(), S, H, own, bdev.data_ptr(), D ** -0.5, work.data_ptr(), need,
                     rows_per_seq=r, out_f32=out_f32)
        ref.done()
        got = f64(out).reshape(n, r, Kv, G, D)
        want, _, gam, mag = ref.attend(f64(q), f64(k), f64(clean), base, r, D ** -0.5)
        tol = ref.bound(gam, mag, cap + 64, want, T, out_f32)
        inf = np.zeros(got.shape)
        inf[odd, hidden:, :, :, 3] = np.inf
        inf[odd, hidden:, 1, :, D - 2] = -np.inf
        seen = ~np.isfinite(inf)
        assert np.array_equal(got[seen], inf[seen])
        off = (np.abs(got.reshape(want.shape) - want) / tol).reshape(got.shape)[~seen]
        assert np.all(off <= 1.0), float(np.nanmax(off))
    assert cuda.last_device_error(0) == 0


def repeats(n, r, H, Kv, D, T, Tp, cap, out_f32, acc, other):
    rng = np.random.default_rng(n + D + cap)
    S = n * r
    q = torch.from_numpy(rng.standard_normal((S, H, D), dtype=np.float32)).to(TYPES[T]).cuda()
    k, v = (ref.cache(rng, n, Kv, cap, D, T) for _ in range(2))
    pk, pv = (ref.cache(rng, 1, Kv, max(Tp, 1), D, T) for _ in range(2))
    base = rng.integers((cap - r) // 2, cap - r + 1, n)
    start = torch.from_numpy(rng.random((n, Kv, cap), dtype=np.float32)).cuda()
    a, bdev = start.clone(), i32(base)
    out = torch.zeros((S, H, D), dtype=torch.float32 if out_f32 else TYPES[T], device="cuda")
    own, pre = ref.view(k, v, T, acc=a if acc else None), ref.view(pk, pv, T)
    need = at.attention_workspace(0, S, H, own, Tp, r)
    work, first = torch.zeros(need, dtype=torch.uint8, device="cuda"), None
    for fill in (0, 255, 63):
        work.fill_(fill), other.fill_(fill), a.copy_(start), out.fill_(1000.0)
        torch.cuda.synchronize()
        at.attention(0, out.data_ptr(), q.data_ptr(), S, H, own, bdev.data_ptr(), D ** -0.5, work.data_ptr(), need,
                     rows_per_seq=r, prefix=pre if Tp else None, prefix_len=Tp, out_f32=out_f32)
        ref.done()
        got = out.view(torch.int32 if out_f32 else torch.int16).clone(), a.view(torch.int32).clone()
        assert bool((out.abs() < 100.0).all())  # all of it was written, and is finite
        assert torch.equal(got[0], (first or got)[0]) and torch.equal(got[1], (first or got)[1]), (n, r, H, Kv, D, T, Tp, cap)
        first = first or got
    assert acc != torch.equal(a, start)
    assert cuda.last_device_error(0) == 0


@pytest.fixture(scope="module")
def other():
    """Memory of more than the last cache's size: filled, it leaves nothing of a call's there."""
    return torch.zeros(1 << 28, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("n, r, H, Kv, D, T, Tp, cap, out_f32, acc", [
    (1, 1, 4, 2, 64, "bf16", 0, 20000, True, True),       # one line of tiles over many CTAs
    (3, 1, 8, 2, 128, "f16", 70, 900, False, False),
    (2, 4, 6, 2, 256, "bf16", 129, 500, True, True),      # 12 row vectors a problem
    (9, 1, 24, 2, 64, "f16", 1500, 400, True, True),      # the prefix on tensor memory, own slots not
    (41, 1, 64, 2, 128, "bf16", 700, 140, False, True),   # a warp joins a row vector
    (2, 40, 32, 2, 64, "bf16", 300, 800, True, True),     # all on tensor memory, weights of many row vectors
    (5, 9, 16, 4, 256, "f16", 0, 300, False, False),
])
def test_attention_repeats_its_bits(dev, other, n, r, H, Kv, D, T, Tp, cap, out_f32, acc):
    """The same bits from the same inputs, whatever output, scratch and the chip's caches held before."""
    repeats(n, r, H, Kv, D, T, Tp, cap, out_f32, acc, other)


@pytest.mark.parametrize("D, T", [(64, "bf16"), (64, "f16"), (128, "bf16"), (128, "f16"), (256, "bf16"), (256, "f16")])
def test_attention_repeats_its_bits_over_its_ranges(dev, other, D, T):
    rng = np.random.default_rng(D + len(T))
    for t in range(24):
        n, r = [(int(rng.integers(1, 40)), 1), (int(rng.integers(1, 6)), int(rng.integers(2, 17))),
                (1, int(rng.integers(17, 65)))][t % 3]
        Kv = int(rng.integers(1, 4))
        Tp, cap = (int(np.exp(rng.uniform(0, np.log(2000)))) for _ in range(2))
        repeats(n, r, Kv * int(rng.integers(1, 11)), Kv, D, T, Tp * (t & 1), cap + r, t % 4 < 2, t % 5 < 3, other)


@pytest.mark.parametrize("G, r, Tp", [(4, 1, 0), (3, 4, 0), (16, 1, 700), (4, 9, 0), (20, 1, 500)])
@pytest.mark.parametrize("T", ["f16", "bf16"])
def test_small_weights_beside_a_large_one(dev, T, G, r, Tp):
    """One key takes most of the weight, 12000 others the same small share w each: what the rounding of w to 16-bit terms
    loses is lost 12000 times over.  With an fp32 output that is up to 2^-21 w, and from an f16 cache 2^-30 of the
    largest weight besides (f16's smallest step, behind the factor 2^6)."""
    D, cap = 64, 12000
    rng = np.random.default_rng(G)
    k = torch.zeros((1, 1, cap, D), dtype=TYPES[T], device="cuda")
    k[..., 0] = -1.0
    k[:, :, 7, 0] = 0.0
    v = torch.from_numpy(rng.random((1, 1, cap, D), dtype=np.float32) + 0.5).to(TYPES[T]).cuda()
    v[..., ::2], v[:, :, 7] = 1.0, 0.0
    pk, pv = k[:, :, 50:50 + max(Tp, 1)].contiguous(), v[:, :, 50:50 + max(Tp, 1)].contiguous()
    base, scale = cap - r, np.float32(np.log(2.0))
    own, pre, bdev = ref.view(k, v, T), ref.view(pk, pv, T), i32([base])
    need = at.attention_workspace(0, r, G, own, Tp, r)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    q, out = torch.zeros((r, G, D), dtype=TYPES[T], device="cuda"), torch.zeros((r, G, D), device="cuda")
    sums = np.cumsum(f64(v)[0, 0], 0)[base:] + (f64(pv)[0, 0].sum(0) if Tp else 0.0)  # of the values row i sees
    count = base + np.arange(r)[:, None] + (Tp if Tp else 0)                          # small weights row i sees
    for x in np.linspace(6.0, 24.0, 73):
        q[..., 0] = float(x)
        torch.cuda.synchronize()
        at.attention(0, out.data_ptr(), q.data_ptr(), r, G, own, bdev.data_ptr(), float(scale), work.data_ptr(), need,
                     rows_per_seq=r, prefix=pre if Tp else None, prefix_len=Tp)
        ref.done()
        w = np.exp(-float(q[0, 0, 0]) * float(scale))
        want = (w * sums / (1.0 + w * count))[:, None, :]
        # Scores are one product each: two roundings of the scale and two of a score of up to 24 (half a step of 2^-19), to
        # base e; 2^-22 of the exponential; both for weight and sum.  A CTA has up to 4 tiles here, 48 matrix
        # instructions that add to a sum, two fp32 roundings each; up to 148 partial results follow.
        each = 2 * (np.log(2.0) * (24 * 2.0 ** -23 + 2.0 ** -19) + 2.0 ** -22) + 48 * 2.0 ** -23 + 148 * 2.0 ** -24
        tiny = 1.5 * count[:, :, None] * 2.0 ** -30 if T == "f16" else 0.0
        off = np.abs(f64(out) - want)
        assert np.all(off <= want * (each + 2.0 ** -21) + tiny), (x, float((off / want).max()))


@pytest.mark.parametrize("n, r, G, Kv, D, T, Tp, out_f32", [
    (3, 1, 4, 2, 64, "bf16", 150, True), (2, 3, 4, 2, 128, "f16", 0, False), (5, 9, 4, 1, 256, "bf16", 0, True),
    (4, 12, 12, 2, 64, "f16", 90, True), (24, 1, 8, 2, 128, "bf16", 400, False), (1, 40, 5, 2, 128, "bf16", 70, True),
])
def test_infinite_values_stay_in_the_elements_that_see_them(dev, n, r, G, Kv, D, T, Tp, out_f32):
    """In the prefix, among the slots that all rows of a sequence see, and among the new ones, of which masks hide some."""
    rng = np.random.default_rng(n + D)
    H, S, cap = G * Kv, n * r, r + 150
    q = torch.from_numpy(rng.standard_normal((S, H, D), dtype=np.float32)).to(TYPES[T]).cuda()
    k, v = (ref.cache(rng, n, Kv, cap, D, T) for _ in range(2))
    pk, pv = (ref.cache(rng, 1, Kv, max(Tp, 1), D, T) for _ in range(2))
    base = rng.integers(1, cap - r + 1, n)
    bits = rng.integers(0, 1 << min(r, 62), S).astype(np.uint64)
    odd = np.array([np.inf, -np.inf, np.nan])
    for b in range(n):
        for _ in range(3):
            low = 0 if rng.random() < 0.4 else base[b]
            v[b, rng.integers(Kv), rng.integers(low, base[b] + r), rng.integers(D)] = float(rng.choice(odd))
        k[b, :, base[b] + r:], v[b, :, base[b] + r:] = float("nan"), float("-inf")
    if Tp:
        pv[0, 0, rng.integers(Tp), 5] = float("inf")
    clean, pclean = (torch.where(torch.isfinite(x), x, 0.0) for x in (v, pv))
    out = torch.zeros((S, H, D), dtype=torch.float32 if out_f32 else TYPES[T], device="cuda")
    own, pre, bdev, mask = ref.view(k, v, T), ref.view(pk, pv, T), i32(base), torch.from_numpy(bits.view(np.int64)).cuda()
    need = at.attention_workspace(0, S, H, own, Tp, r)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    at.attention(0, out.data_ptr(), q.data_ptr(), S, H, own, bdev.data_ptr(), D ** -0.5, work.data_ptr(), need, rows_per_seq=r,
                 prefix=pre if Tp else None, prefix_len=Tp, mask=mask.data_ptr(), out_f32=out_f32)
    ref.done()
    got, prefix = f64(out), (f64(pk)[0], f64(pclean)[0]) if Tp else (None, None)
    want, _, gam, mag = ref.attend(f64(q), f64(k), f64(clean), base, r, D ** -0.5, *prefix, mask=bits)
    tol = ref.bound(gam, mag, Tp + cap + 64, want, T, out_f32)
    hit = np.zeros((S, Kv, D), bool)  # what an odd value is seen by
    for s in range(S):
        seen = ref.visible(cap, base[s // r], s % r, r, bits[s])
        hit[s] = (~np.isfinite(f64(v[s // r])) & seen[None, :, None]).any(1)
        if Tp:
            hit[s] |= (~np.isfinite(f64(pv[0]))).any(1)
    hit = np.repeat(hit, G, 1)
    assert hit.any() and np.array_equal(~np.isfinite(got), hit)
    assert np.all((np.abs(got - want) <= tol)[~hit])
