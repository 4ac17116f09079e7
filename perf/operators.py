"""The attention half of a decode layer, as cases that can be prepared, run and checked.

Three operators around one cache of keys and values (16-bit values, ``[sequence, kv head, slot, dim]``):

* ``norm``   query and key norms per head, the rotation of both and the store of keys and values into the cache,
             in one pass over the projection's fp32 rows (``attention.qk_norm_rope``);
* ``attn``   attention of a batch whose sequences share a long prefix, each with slots of its own behind it, one or
             several rows a sequence (``attention.attention``);
* ``evict``  the slots of a cache that received the most attention, moved into a smaller one
             (``attention.kv_evict``).

With ``own`` set, ``run`` calls the framework; otherwise it computes the same in elementary torch operations, in
32 bits (angles in 64), rounded once.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = 0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
THETA = 10000.0
EPS = 1e-6


def listed():
    return [
        # one new token of one sequence (hidden 6144 as 48 heads of 128): pure latency
        dict(name="norm_decode_1", kind="norm", n=1, r=1, H=48, Kv=8, D=128, R=128, style=0, T="bf16", cap=256,
             norm=True, far=9000, pad=0, slot_major=False),
        # 8-node drafts of 33 sequences far into a context: part of the head rotates, halves instead of pairs
        dict(name="norm_verify_33x8", kind="norm", n=33, r=8, H=20, Kv=4, D=256, R=64, style=1, T="f16", cap=64,
             norm=True, far=900000, pad=12, slot_major=True),
        # a prompt chunk, and the longest one, straight into the shared prefix
        dict(name="norm_prompt_1000", kind="norm", n=1, r=1000, H=32, Kv=32, D=64, R=64, style=0, T="bf16", cap=1000,
             norm=False, far=0, pad=0, slot_major=False),
        dict(name="norm_prompt_4096", kind="norm", n=1, r=4096, H=48, Kv=8, D=128, R=128, style=0, T="bf16", cap=4096,
             norm=True, far=0, pad=0, slot_major=False),
        # one token of one young sequence without a prefix: latency
        dict(name="attn_decode_1", kind="attn", n=1, r=1, H=48, Kv=8, D=128, Tp=0, cap=300, T="bf16", out="f32",
             acc=False, tree=False, slot_major=False),
        # a decode batch of 32 behind a common system prompt; the weights are kept for the eviction
        dict(name="attn_batch_32", kind="attn", n=32, r=1, H=48, Kv=8, D=128, Tp=8192, cap=1024, T="bf16", out="f32",
             acc=True, tree=False, slot_major=False),
        # the longest prefix, a group of eight query heads a key head
        dict(name="attn_prefix_32768", kind="attn", n=32, r=1, H=64, Kv=8, D=128, Tp=32768, cap=2048, T="bf16",
             out="16", acc=False, tree=False, slot_major=False),
        # verification of 8-node draft trees: every row sees its own ancestors
        dict(name="attn_verify_5x8", kind="attn", n=5, r=8, H=28, Kv=4, D=64, Tp=2001, cap=4000, T="f16", out="f32",
             acc=False, tree=True, slot_major=True),
        # two long contexts of their own, no prefix: the split over one long axis
        dict(name="attn_long_2", kind="attn", n=2, r=1, H=32, Kv=8, D=128, Tp=0, cap=50000, T="bf16", out="f32",
             acc=True, tree=False, slot_major=False),
        # a 64-row chunk of a prompt behind what is already cached, wide heads
        dict(name="attn_chunk_64", kind="attn", n=1, r=64, H=16, Kv=2, D=256, Tp=0, cap=6000, T="f16", out="16",
             acc=False, tree=False, slot_major=False),
        # a full budget of one sequence, a few slots over: the eviction inside a decode loop
        dict(name="evict_step_1", kind="evict", n=1, Kv=8, D=128, cap=544, keep=512, sinks=4, recent=32, T="bf16"),
        # prompts of a batch brought down to a budget
        dict(name="evict_prompt_6", kind="evict", n=6, Kv=8, D=128, cap=40000, keep=2048, sinks=4, recent=256,
             T="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _drawn(rng):
    kind = rng.choice(["norm"] * 3 + ["attn"] * 5 + ["evict"] * 3)
    T, D, Kv = rng.choice(["bf16", "f16"]), rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 5, 8, 8])
    if kind == "norm":
        r = rng.choice([1, 1, _log_int(rng, 2, 64), 0])
        n = _log_int(rng, 1, 64) if r else 1
        r = r or _log_int(rng, 65, 4096)
        return dict(kind="norm", n=n, r=r, H=Kv * rng.randint(1, 10), Kv=Kv, D=D, R=rng.choice([D, D, D // 2, D - 2]),
                    style=rng.randint(0, 1), T=T, cap=r + rng.randint(0, 40), norm=rng.random() < 0.8,
                    far=rng.choice([0, 0, _log_int(rng, 1, 1000000)]), pad=4 * rng.randint(0, 5),
                    slot_major=rng.random() < 0.4)
    if kind == "attn":
        n, r = rng.choice([(_log_int(rng, 1, 64), 1)] * 3 + [(rng.randint(1, 8), rng.randint(2, 16)),
                                                            (1, rng.randint(17, 64))])
        return dict(kind="attn", n=n, r=r, H=Kv * rng.randint(1, 12), Kv=Kv, D=D,
                    Tp=rng.choice([0, _log_int(rng, 16, 32768), _log_int(rng, 16, 32768)]),
                    cap=r + _log_int(rng, 1, 50000 if n < 4 else 4000), T=T, out=rng.choice(["f32", "f32", "16"]),
                    acc=rng.random() < 0.4, tree=r > 1 and rng.random() < 0.5, slot_major=rng.random() < 0.3)
    keep = _log_int(rng, 16, 8000)
    return dict(kind="evict", n=rng.randint(1, 8), Kv=Kv, D=D, cap=keep + _log_int(rng, 1, 40000), keep=keep,
                sinks=rng.randint(0, 8), recent=rng.randint(0, keep // 2), T=T)


def draw(rng: random.Random):
    most = [work(c) for c in listed()]
    while True:
        c = _drawn(rng)
        w = work(c)
        if any(w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"] for m in most):
            return c


# ------------------------------------------------------------------------------------ inputs
def _lengths(case, least):
    """The slots in use of every sequence, the first one full: they belong to the case, the values to the seed."""
    lens = np.random.default_rng(case["n"] * 7 + case["cap"]).integers(max(least, case["cap"] // 4), case["cap"] + 1,
                                                                      case["n"])
    lens[0] = case["cap"]
    return lens.astype(np.int32)


def _cache(gen, n, Kv, cap, D, T, slot_major):
    """Keys or values [n, Kv, cap, D] in either order of memory."""
    t = torch.randn((n, cap, Kv, D) if slot_major else (n, Kv, cap, D), generator=gen, device=gen.device)
    t = t.to(TYPES[T])
    return t.transpose(1, 2) if slot_major else t


def _inputs(case, seed):
    dev = torch.device("cuda:%d" % DEV)
    gen = torch.Generator(dev).manual_seed(seed)
    kind, n, Kv, D, T = case["kind"], case["n"], case["Kv"], case["D"], case["T"]
    s = dict(case=case)
    if kind == "evict":
        lens = _lengths(case, case["keep"] // 2)
        s["len"] = torch.from_numpy(lens).to(dev)
        s["k"] = _cache(gen, n, Kv, case["cap"], D, T, False)
        s["v"] = _cache(gen, n, Kv, case["cap"], D, T, False)
        # weights of earlier steps have a heavy tail; positions have gaps where earlier slots went
        s["acc"] = torch.exp(2.0 * torch.randn((n, Kv, case["cap"]), generator=gen, device=dev))
        gaps = torch.randint(1, 4, (n, Kv, case["cap"]), generator=gen, device=dev)
        s["pos"] = (torch.cumsum(gaps, 2) - gaps[:, :, :1]).to(torch.int32)
        return s
    r, H = case["r"], case["H"]
    rows = n * r
    if kind == "norm":
        width = (H + 2 * Kv) * D
        s["qkv"] = 1.5 * torch.randn((rows, width + case["pad"]), generator=gen, device=dev)
        s["wq"] = 1.0 + 0.1 * torch.randn(D, generator=gen, device=dev)
        s["wk"] = 1.0 + 0.1 * torch.randn(D, generator=gen, device=dev)
        s["k"] = _cache(gen, n, Kv, case["cap"], D, T, case["slot_major"])
        s["v"] = _cache(gen, n, Kv, case["cap"], D, T, case["slot_major"])
        s["slots"] = torch.full((n, Kv, case["cap"]), -1, dtype=torch.int32, device=dev)
        s["base"] = torch.randint(0, case["cap"] - r + 1, (n,), generator=gen, device=dev).to(torch.int32)
        at = s["base"][:, None] + torch.arange(r, device=dev, dtype=torch.int32)
        s["pos"] = (at + case["far"]).reshape(-1).to(torch.int32)
        return s
    s["q"] = (2.0 * torch.randn((rows, H, D), generator=gen, device=dev)).to(TYPES[T])
    if case["Tp"]:
        s["pk"] = _cache(gen, 1, Kv, case["Tp"], D, T, case["slot_major"])
        s["pv"] = _cache(gen, 1, Kv, case["Tp"], D, T, case["slot_major"])
    s["k"] = _cache(gen, n, Kv, case["cap"], D, T, case["slot_major"])
    s["v"] = _cache(gen, n, Kv, case["cap"], D, T, case["slot_major"])
    s["base"] = torch.from_numpy(_lengths(case, r) - np.int32(r)).to(dev)
    if case["tree"]:  # every node's parent is an earlier node of its tree
        bits, tree = np.zeros((n, r), np.int64), np.random.default_rng(seed)
        for i in range(r):
            up = tree.integers(0, i, n) if i else None
            bits[:, i] = (bits[np.arange(n), up] if i else 0) | (np.int64(1) << np.int64(i))
        s["mask"] = torch.from_numpy(bits.reshape(-1)).to(dev)
    if case["acc"]:
        s["acc"] = torch.rand((n, Kv, case["cap"]), generator=gen, device=dev)
    return s


# ----------------------------------------------------------------------------------- prepare, run
def _view(at, k, v, T, pos=None, acc=None):
    n, Kv, cap, D = k.shape
    return at.KvView(k.data_ptr(), v.data_ptr(), n, Kv, cap, D, T, pos=0 if pos is None else pos.data_ptr(),
                     acc=0 if acc is None else acc.data_ptr(), strides=k.stride()[:3])


def prepare(case, seed):
    s = _inputs(case, seed)
    dev, kind, T = s["k"].device, case["kind"], case["T"]
    rows = case["n"] * case.get("r", 0)
    if kind == "norm":
        s["q"] = torch.zeros((rows, case["H"], case["D"]), dtype=TYPES[T], device=dev)
    elif kind == "attn":
        s["out"] = torch.zeros((rows, case["H"], case["D"]), device=dev,
                               dtype=torch.float32 if case["out"] == "f32" else TYPES[T])
    else:
        shape = (case["n"], case["Kv"], case["keep"])
        s["dk"], s["dv"] = (torch.zeros(shape + (case["D"],), dtype=TYPES[T], device=dev) for _ in range(2))
        s["dpos"], s["index"] = (torch.zeros(shape, dtype=torch.int32, device=dev) for _ in range(2))
        s["dacc"] = torch.zeros(shape, device=dev)
        s["dlen"] = torch.zeros(case["n"], dtype=torch.int32, device=dev)
    if own:
        from peregrine_b200 import attention as at, cuda

        if cuda.device_count() == 0 and cuda.init([DEV]) < 1:
            raise RuntimeError("the backend could not initialise its device")
        s["at"] = at
        if kind == "norm":
            s["kv"] = _view(at, s["k"], s["v"], T, pos=s["slots"])
        elif kind == "attn":
            s["kv"] = _view(at, s["k"], s["v"], T, acc=s.get("acc"))
            s["prefix"] = _view(at, s["pk"], s["pv"], T) if case["Tp"] else None
            need = at.attention_workspace(DEV, rows, case["H"], s["kv"], case["Tp"], case["r"])
            s["work"] = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        else:
            s["kv"] = _view(at, s["k"], s["v"], T, s["pos"], s["acc"])
            s["to"] = _view(at, s["dk"], s["dv"], T, s["dpos"], s["dacc"])
    torch.cuda.synchronize()  # the backend works on a stream of its own
    return s


def _plain_norm(s):
    c = s["case"]
    n, r, H, Kv, D, R = (c[x] for x in ("n", "r", "H", "Kv", "D", "R"))
    x = s["qkv"][:, :(H + 2 * Kv) * D].reshape(n, r, H + 2 * Kv, D)
    q, k, v = x[:, :, :H], x[:, :, H:H + Kv], x[:, :, H + Kv:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["wq"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["wk"]
    j = torch.arange(R // 2, device=x.device, dtype=torch.float64)
    angle = s["pos"].reshape(n, r, 1, 1).double() * torch.pow(THETA, -2.0 * j / R)
    cs, sn = torch.cos(angle).float(), torch.sin(angle).float()

    def rotate(t):
        a, b = (t[..., :R:2], t[..., 1:R:2]) if c["style"] == 0 else (t[..., :R // 2], t[..., R // 2:R])
        return torch.cat([a * cs - b * sn, b * cs + a * sn, t[..., R:]], -1)

    s["q"].copy_(rotate(q).reshape(n * r, H, D))
    seq = torch.arange(n, device=x.device)[:, None]
    slot = s["base"][:, None].long() + torch.arange(r, device=x.device)
    s["k"][seq, :, slot] = rotate(k).to(s["k"].dtype)
    s["v"][seq, :, slot] = v.to(s["v"].dtype)
    s["slots"][seq, :, slot] = s["pos"].reshape(n, r, 1).expand(n, r, Kv)
    return {"q": s["q"], "k": s["k"], "v": s["v"], "slots": s["slots"]}


def _plain_attn(s):
    c = s["case"]
    n, r, H, Kv, D, cap = (c[x] for x in ("n", "r", "H", "Kv", "D", "cap"))
    q = s["q"].float().reshape(n, r, Kv, H // Kv, D) * (D ** -0.5)
    t = torch.arange(cap, device=q.device)[None, None, :] - s["base"][:, None, None]
    if c["tree"]:
        bit = s["mask"].reshape(n, r, 1) >> t.clamp(0, r - 1) & 1
        seen = (t < 0) | ((t < r) & (bit == 1))
    else:
        seen = t <= torch.arange(r, device=q.device)[None, :, None]
    seen = seen[:, :, None, None, :]
    sc = torch.einsum("nrhgd,nhtd->nrhgt", q, s["k"].float()).masked_fill(~seen, -math.inf)
    if c["Tp"]:
        sc = torch.cat([torch.einsum("nrhgd,htd->nrhgt", q, s["pk"][0].float()), sc], -1)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.einsum("nrhgt,nhtd->nrhgd", p[..., c["Tp"]:], s["v"].float())
    if c["Tp"]:
        o = o + torch.einsum("nrhgt,htd->nrhgd", p[..., :c["Tp"]], s["pv"][0].float())
    s["out"].copy_(o.reshape(n * r, H, D))
    if not c["acc"]:
        return s["out"]
    s["acc"] += p[..., c["Tp"]:].sum((1, 3))
    return {"out": s["out"], "acc": s["acc"]}


def _plain_evict(s):
    c = s["case"]
    n, Kv, D, cap, keep = (c[x] for x in ("n", "Kv", "D", "cap", "keep"))
    i = torch.arange(cap, device=s["k"].device)
    used = (i < s["len"][:, None, None]).expand(n, Kv, cap)
    last = s["pos"].masked_fill(~used, -1).amax(-1, keepdim=True)
    first = (s["pos"] < c["sinks"]) | (s["pos"] > last - c["recent"])
    key = torch.where(first, 1e300, s["acc"].double()).masked_fill(~used, -1.0)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    kept = torch.zeros_like(used).scatter(-1, order[..., :keep], True) & used
    count = torch.clamp(s["len"], max=keep)
    low, j = kept[..., :keep], i[:keep]
    there = j < count[:, None, None]
    moved = kept & (i >= keep)
    table = torch.zeros((n, Kv, cap + 1), dtype=torch.int64, device=i.device)
    rank = torch.where(moved, torch.cumsum(moved, -1) - 1, cap)
    table.scatter_(-1, rank, i.expand(n, Kv, cap))
    hole = torch.cumsum(~low, -1) - 1
    src = torch.where(low, j, torch.gather(table, -1, hole.clamp(min=0)))
    s["index"].copy_(torch.where(there, src, -1))
    s["dlen"].copy_(count)
    src = torch.where(there, src, 0)
    for to, of in (("dpos", "pos"), ("dacc", "acc")):
        s[to].copy_(torch.where(there, torch.gather(s[of], -1, src), s[to]))
    rows = src[..., None].expand(n, Kv, keep, D)
    for to, of in (("dk", "k"), ("dv", "v")):
        s[to].copy_(torch.where(there[..., None], torch.gather(s[of], 2, rows), s[to]))
    return _evicted(s)


def _evicted(s):
    return {"k": s["dk"], "v": s["dv"], "pos": s["dpos"], "acc": s["dacc"], "index": s["index"], "len": s["dlen"]}


def run(s):
    c = s["case"]
    if not own:
        return {"norm": _plain_norm, "attn": _plain_attn, "evict": _plain_evict}[c["kind"]](s)
    at = s["at"]
    if c["kind"] == "norm":
        at.qk_norm_rope(DEV, s["q"].data_ptr(), s["qkv"].data_ptr(), c["n"] * c["r"], c["H"], s["kv"],
                        s["base"].data_ptr(), s["pos"].data_ptr(), THETA, rotary=c["R"], style=c["style"],
                        q_weight=s["wq"].data_ptr() if c["norm"] else 0, k_weight=s["wk"].data_ptr() if c["norm"] else 0,
                        eps=EPS, rows_per_seq=c["r"], row_stride=s["qkv"].stride(0))
        return {"q": s["q"], "k": s["k"], "v": s["v"], "slots": s["slots"]}
    if c["kind"] == "attn":
        at.attention(DEV, s["out"].data_ptr(), s["q"].data_ptr(), c["n"] * c["r"], c["H"], s["kv"],
                     s["base"].data_ptr(), c["D"] ** -0.5, s["work"].data_ptr(), s["work"].numel(),
                     rows_per_seq=c["r"], prefix=s["prefix"], prefix_len=c["Tp"],
                     mask=s["mask"].data_ptr() if c["tree"] else 0, out_f32=c["out"] == "f32")
        return {"out": s["out"], "acc": s["acc"]} if c["acc"] else s["out"]
    at.kv_evict(DEV, s["to"], s["kv"], s["len"].data_ptr(), s["dlen"].data_ptr(), s["index"].data_ptr(), c["keep"],
                sinks=c["sinks"], recent=c["recent"])
    return _evicted(s)


# ---------------------------------------------------------------------------------------- work
def work(case):
    kind, n, Kv, D = case["kind"], case["n"], case["Kv"], case["D"]
    if kind == "norm":
        rows = n * case["r"]
        values = rows * (case["H"] + 2 * Kv) * D
        return {"bytes": float(values * 6 + rows * 4 + rows * Kv * 4), "flops": float(8 * values)}
    if kind == "evict":
        lens = _lengths(case, case["keep"] // 2).astype(np.int64)
        kept = int(np.minimum(lens, case["keep"]).sum()) * Kv
        return {"bytes": float(int(lens.sum()) * Kv * 8 + kept * (2 * (4 * D + 8) + 4)),
                "flops": float(int(lens.sum()) * Kv)}
    rows, lens = n * case["r"], int(_lengths(case, case["r"]).astype(np.int64).sum())
    b = 4 * D * Kv * (case["Tp"] + lens) + rows * case["H"] * D * (2 + (4 if case["out"] == "f32" else 2))
    b += 8 * Kv * lens if case["acc"] else 0
    return {"bytes": float(b), "flops": float(4 * case["H"] * D * (rows * case["Tp"] + case["r"] * lens))}


# --------------------------------------------------------------------------------------- exact
def _exact_evict(case, s):
    """The moves one by one, from the ranking: protected slots, then the larger weight, then the lower slot."""
    n, Kv, D, keep = case["n"], case["Kv"], case["D"], case["keep"]
    lens, pos, acc = s["len"].cpu().numpy(), s["pos"].cpu().numpy(), s["acc"].double().cpu().numpy()
    got = {"k": torch.zeros((n, Kv, keep, D), dtype=torch.float64, device=s["k"].device), "index": None, "len": None}
    got["v"] = torch.zeros_like(got["k"])
    got["acc"], got["pos"] = np.zeros((n, Kv, keep)), None
    for b in range(n):
        for h in range(Kv):
            p, a = pos[b, h, :lens[b]].astype(np.int64), acc[b, h, :lens[b]]
            other = ~((p < case["sinks"]) | (p > p.max() - case["recent"]))
            best = np.lexsort((np.arange(len(p)), -a, other))[:keep]
            src = np.arange(len(best))
            src[np.setdiff1d(src, best)] = np.sort(best[best >= len(src)])
            at = torch.from_numpy(src).to(s["k"].device)
            got["k"][b, h, :len(src)] = s["k"][b, h, at].double()
            got["v"][b, h, :len(src)] = s["v"][b, h, at].double()
            got["acc"][b, h, :len(src)] = a[src]
    return got


def exact(case, seed):
    s = _inputs(case, seed)
    kind, n, Kv, D = case["kind"], case["n"], case["Kv"], case["D"]
    if kind == "evict":
        return _exact_evict(case, s)
    r, H = case["r"], case["H"]
    if kind == "norm":
        x = s["qkv"].double()
        half = case["R"] // 2
        j = torch.arange(half, device=x.device, dtype=torch.float64)
        turn = torch.polar(torch.ones(n * r, half, device=x.device, dtype=torch.float64),
                           s["pos"].double()[:, None] * torch.exp(-j * (2.0 * math.log(THETA) / case["R"])))[:, None, :]

        def head(t, w):
            t = t.reshape(n * r, -1, D)
            if case["norm"]:
                t = t / torch.sqrt((t * t).sum(-1, keepdim=True) / D + EPS) * w.double()
            z = t[..., :2 * half]
            z = torch.view_as_complex(z.reshape(n * r, -1, half, 2).contiguous()) if case["style"] == 0 else \
                torch.complex(z[..., :half], z[..., half:])
            z = z * turn
            return torch.cat([z.real, z.imag, t[..., 2 * half:]], -1)

        q = head(x[:, :H * D], s["wq"])
        k = head(x[:, H * D:(H + Kv) * D], s["wk"])
        v = x[:, (H + Kv) * D:(H + 2 * Kv) * D].reshape(n * r, Kv, D)
        ks, vs = s["k"].double(), s["v"].double()
        for b in range(n):
            at = int(s["base"][b])
            ks[b, :, at:at + r] = k[b * r:(b + 1) * r].transpose(0, 1)
            vs[b, :, at:at + r] = v[b * r:(b + 1) * r].transpose(0, 1)
        return {"q": q, "k": ks, "v": vs, "slots": None}
    out = torch.empty((n, r, H, D), dtype=torch.float64, device=s["k"].device)
    acc = s["acc"].double() if case["acc"] else None
    Tp, G = case["Tp"], H // Kv
    for b in range(n):
        at = int(s["base"][b])
        for h in range(Kv):
            k, v = s["k"][b, h, :at + r].double(), s["v"][b, h, :at + r].double()
            if Tp:
                k, v = torch.cat([s["pk"][0, h].double(), k]), torch.cat([s["pv"][0, h].double(), v])
            q = s["q"].reshape(n, r, H, D)[b, :, h * G:(h + 1) * G].double()
            e = q.reshape(r * G, D) @ k.T / math.sqrt(D)
            e = e.reshape(r, G, -1)
            new = torch.ones((r, r), dtype=torch.bool, device=k.device).tril()
            if case["tree"]:
                m = s["mask"].reshape(n, r)[b]
                new = (m[:, None] >> torch.arange(r, device=k.device)[None, :]) % 2 == 1
            e[:, :, Tp + at:] = torch.where(new[:, None, :], e[:, :, Tp + at:], torch.full_like(e[:, :, Tp + at:], -math.inf))
            w = torch.softmax(e, -1)
            out[b, :, h * G:(h + 1) * G] = (w.reshape(r * G, -1) @ v).reshape(r, G, D)
            if acc is not None:
                acc[b, h, :at + r] += w[:, :, Tp:].sum((0, 1))
    out = out.reshape(n * r, H, D)
    return out if acc is None else {"out": out, "acc": acc}
