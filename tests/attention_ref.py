"""Plain 64-bit forms of the attention operators, in numpy, and device buffers for their tests."""
import numpy as np
import torch

from peregrine_b200 import attention as at, cuda

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step relative to the value (eps / 2 of the type)


def f64(t):
    return t.detach().cpu().double().numpy()


def cache(rng, n, Kv, cap, D, T, slot_major=False, std=1.0):
    x = torch.from_numpy(rng.standard_normal((n, cap, Kv, D) if slot_major else (n, Kv, cap, D), dtype=np.float32) * std)
    x = x.to(TYPES[T]).cuda()
    return x.transpose(1, 2) if slot_major else x


def view(k, v, T, pos=None, acc=None):
    n, Kv, cap, D = k.shape
    return at.KvView(k.data_ptr(), v.data_ptr(), n, Kv, cap, D, T, pos=0 if pos is None else pos.data_ptr(),
                     acc=0 if acc is None else acc.data_ptr(), strides=k.stride()[:3])


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def done():
    """Both sides meet: torch's stream and the backend's."""
    assert cuda.lib().coli_cuda_pipe_sync(0) == 1
    torch.cuda.synchronize()


def visible(n_slots, base, i, r, bits):
    """Own slots that row i sees, as a truth value per slot."""
    t = np.arange(n_slots)
    new = t - base
    ok = (new >= 0) & (new < r)
    pick = np.array([(int(bits) >> int(j)) & 1 if 0 <= j < 64 else 0 for j in new], bool) if bits is not None else new <= i
    return (t < base) | (ok & pick)


def attend(q, k, v, base, r, scale, pk=None, pv=None, mask=None):
    """out [S, H, D], weights added per own slot [n, Kv, cap], and the bound gamma, sum p |v| of its error."""
    S, H, D = q.shape
    n, Kv, cap, _ = k.shape
    G = H // Kv
    out, mag, gam = np.zeros((S, H, D)), np.zeros((S, H, D)), np.zeros((S, H, 1))
    acc = np.zeros((n, Kv, cap))
    for b in range(n):
        if base[b] < 0:
            continue
        for i in range(r):
            row = b * r + i
            sel = np.nonzero(visible(cap, base[b], i, r, None if mask is None else mask[row]))[0]
            for h in range(H):
                kk, vv = k[b, h // G][sel], v[b, h // G][sel]
                tp = 0
                if pk is not None:
                    tp = pk.shape[1]
                    kk, vv = np.concatenate([pk[h // G], kk]), np.concatenate([pv[h // G], vv])
                if len(kk) == 0:
                    continue
                s = kk @ q[row, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[row, h] = p @ vv
                mag[row, h] = p @ np.abs(vv)
                gam[row, h] = (np.abs(kk) @ np.abs(q[row, h])).max() * abs(scale) * D * 2.0 ** -24 + np.abs(s).max() * 2.0 ** -23
                acc[b, h // G][sel] += p[tp:]
    return out, acc, gam, mag


def bound(gam, mag, terms, out, T, out_f32):
    """A score is a sum of D exact products in fp32 (each step half an ulp of the running sum, so D 2^-24 of the sum
    of magnitudes) and is scaled and taken to base two with two more roundings (`gam`); a weight is off by that,
    2^-21 of the exponential and its split, and weights and sum are off alike, so twice; sums of `terms` products in
    fp32; for 16-bit outputs the weights and the result are each rounded to the type."""
    e = mag * (2 * (gam + 2.0 ** -21) + terms * 2.0 ** -24)
    if not out_f32:
        e = e + mag * HALF[T] + (np.abs(out) + e) * HALF[T] + (2.0 ** -25 if T == "f16" else 0.0)
    return e + 1e-30


def rank_evict(pos, acc, length, keep, sinks, recent):
    """Source slot of every kept one, for one (sequence, kv head)."""
    length = min(length, len(pos))
    p = pos[:length].astype(np.int64)
    if length <= keep:
        return np.arange(length)
    last = p.max()

    def key(t):
        if p[t] < sinks or p[t] > last - recent:
            return (0, 0.0, t)
        a = float(acc[t])
        return (2, 0.0, t) if a != a else (1, -a, t)

    best = np.array(sorted(range(length), key=key)[:keep])
    src = np.arange(keep)
    src[np.setdiff1d(src, best)] = np.sort(best[best >= keep])
    return src
