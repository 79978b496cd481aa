"""Definitions in 64 bits of the bounded-cache operators, with the tolerances
that their arithmetic allows, and the caches their tests read.

Tolerances count, per output: the rounding of the result to fp16 (2^-11
relative), the attention weights rounded to fp16 before the product with V
(2^-11 relative; below 2^-14 of the row's reference maximum an absolute 2^-25,
divided by the row's sum), the scores' fp32 accumulation of D exact products
(D 2^-24 of the sum of their magnitudes), a few fp32 roundings of exponents,
and the fp32 sums over n keys (n 2^-24, the worst order)."""
import math

import numpy as np

from gpu_util import make_block_tables, to_gpu

PAGE = 16
U32 = 2.0 ** -24
U16 = 2.0 ** -11


def visible(p, n, window, sinks):
    """Boolean over keys 0 .. n-1: those the query at position p attends."""
    j = np.arange(n)
    see = j <= p
    if window > 0:
        see &= (j < sinks) | (p - j < window)
    return see


def attend(q, k, v, see):
    """q [G, D], k, v [n, D], see [n]: out [G, D], its tolerance, p [G, n], lse [G],
    and the bound on the scores' error."""
    q, k = q.astype(np.float64), k[see].astype(np.float64)
    v = v[see].astype(np.float64)
    d, n = q.shape[1], k.shape[0]
    s = q @ k.T / math.sqrt(d)
    size = np.abs(q) @ np.abs(k).T / math.sqrt(d)
    ds = (d + 4) * U32 * float(size.max()) + 4 * U32 * float(np.abs(s).max())
    m = s.max(1, keepdims=True)
    e = np.exp(s - m)
    l = e.sum(1, keepdims=True)
    p = e / l
    out = p @ v
    spread = p @ np.abs(v)
    # the reference maximum may lie up to 2^8 below the largest weight
    small = n * 2.0 ** -25 * np.abs(v).max() / l
    tol = U16 * np.abs(out) + (2 * U16 + 2 * ds + 2 * n * U32) * spread + small + 2.0 ** -25
    full = np.zeros((q.shape[0], see.shape[0]))
    full[:, see] = p
    return out, tol, full, (m + np.log(l))[:, 0], ds


class Cache:
    """K and V of `lens` tokens per sequence, in pages or strided, and on the host
    as [B][Hkv][T][D]; what lies outside the sequences is NaN."""

    def __init__(self, rng, lens, hkv, d, paged=True, scale=1.0, cap=None):
        import kvhp
        self.lens = np.asarray(lens, np.int32)
        self.hkv, self.d, self.paged = hkv, d, paged
        B, T = len(self.lens), max(1, int(self.lens.max()))
        self.cap = T if cap is None else cap
        shape = (B, hkv, T, d)
        self.k = (rng.standard_normal(shape) * scale).astype(np.float16)
        self.v = (rng.standard_normal(shape) * scale).astype(np.float16)
        self.kvhp = kvhp
        if paged:
            self.bt, self.pages = make_block_tables(rng, self.lens)

    def upload(self):
        """Tensors and views of the present host arrays."""
        B, _, T, _ = self.k.shape
        if self.paged:
            self.pk, self.pv = (np.full((self.hkv, self.pages, PAGE, self.d), np.nan, np.float16)
                                for _ in range(2))
            for b, n in enumerate(self.lens):
                for i in range((int(n) + PAGE - 1) // PAGE):
                    m = min(PAGE, int(n) - PAGE * i)
                    pid = self.bt[b, i]
                    if pid >= 0:
                        self.pk[:, pid, :m] = self.k[b, :, PAGE * i:PAGE * i + m]
                        self.pv[:, pid, :m] = self.v[b, :, PAGE * i:PAGE * i + m]
            self.pool_k, self.pool_v, self.bt_d = to_gpu(self.pk), to_gpu(self.pv), to_gpu(self.bt)
            self.kv = self.kvhp.paged_view(self.pool_k, self.bt_d)
            self.vv = self.kvhp.paged_view(self.pool_v, self.bt_d)
        else:   # [B][T][Hkv][D], as a projection leaves them
            k, v = self.k.copy(), self.v.copy()
            for b, n in enumerate(self.lens):
                k[b, :, n:], v[b, :, n:] = np.nan, np.nan
            self.pool_k, self.pool_v = (to_gpu(x.transpose(0, 2, 1, 3)) for x in (k, v))
            st = (T * self.hkv * self.d, self.d, self.hkv * self.d)
            self.kv = self.kvhp.strided_view(self.pool_k, *st)
            self.vv = self.kvhp.strided_view(self.pool_v, *st)
        self.lens_d = to_gpu(self.lens)
        return self

    def slots(self, b):
        """(page, slot) of every position of sequence b."""
        j = np.arange(int(self.lens[b]))
        return self.bt[b, j // PAGE], j % PAGE


def workspace(nbytes):
    import torch
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes else None


def decode_ref(q, c, window, sinks):
    """Outputs [B][Hq][D] and tolerances; weights per (b, kvh): sums over the group."""
    B, hq, d = q.shape
    G = hq // c.hkv
    out, tol = np.zeros((B, hq, d)), np.full((B, hq, d), 2.0 ** -25)
    sums, rel = {}, {}
    for b in range(B):
        n = min(int(c.lens[b]), c.cap)
        if n <= 0:
            continue
        see = visible(n - 1, n, window, sinks)
        for h in range(c.hkv):
            hs = slice(h * G, (h + 1) * G)
            o, t, p, _, ds = attend(q[b, hs], c.k[b, h, :n], c.v[b, h, :n], see)
            out[b, hs], tol[b, hs] = o, t
            sums[b, h], rel[b, h] = p.sum(0), 2 * ds + 2 * (n + 16) * U32
    return out, tol, sums, rel


def check(got, ref, tol, what=""):
    got = np.asarray(got, np.float64)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside, first "
                           f"{np.argwhere(bad)[:3].tolist()} got {got[bad][:3]} "
                           f"want {np.asarray(ref)[bad][:3]} tol {np.asarray(tol)[bad][:3]}")


def plan_ref(w, age, n, budget, sinks, recent, newest):
    """Moves [(from, to)] that cut one (sequence, head) of n slots to its budget."""
    if n <= budget:
        return []
    guard = (age[:n] < sinks) | (age[:n].astype(np.int64) > newest - recent)
    w = w[:n].astype(np.float64)
    # NaN below everything, protected slots above; equal: the lowest slot
    level = np.where(guard, 2, np.where(np.isnan(w), 0, 1))
    w = np.where(level == 1, w, 0.0)
    order = sorted(range(n), key=lambda j: (-level[j], -w[j], j))
    keep = np.zeros(n, bool)
    keep[order[:budget]] = True
    src = [j for j in range(budget, n) if keep[j]]
    dst = [j for j in range(budget) if not keep[j]]
    assert len(src) == len(dst)
    return list(zip(src, dst))
