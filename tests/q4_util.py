"""The 4-bit cache's format in numpy, caches for its tests, and the rotation in 64
bits.

A row's scale and offset are computed in fp32, each step rounded as IEEE says, so
codes and numbers are equal bits, not near ones.  Attention over what the rows
stand for is held to bounded_util's tolerances: s and n + r are exact operands, so
nothing but the score's sum, the weight's one rounding to fp16 and the result's
differ from 64 bits."""
import numpy as np

from bounded_util import PAGE, U16, U32, attend, check   # noqa: F401
from gpu_util import make_block_tables, to_gpu

NAN_ROW = 0x7e00


def quantise(x):
    """fp16 rows [..., D]: codes uint8 [..., D] and (s, r) fp16 [..., 2]."""
    x = np.asarray(x, np.float16)
    f = x.astype(np.float32)
    bad = ~np.isfinite(f).all(-1, keepdims=True)
    f = np.where(bad, np.float32(0), f)
    lo, hi = f.min(-1, keepdims=True) + np.float32(0), f.max(-1, keepdims=True)   # no -0
    flat = lo == hi
    t = np.maximum((hi - lo) * (np.float32(1) / np.float32(15)),
                   np.maximum(np.abs(lo), np.abs(hi)) * (np.float32(1) / np.float32(1984)))
    s = t.astype(np.float16)
    s = np.where(s.astype(np.float32) < t, (s.view(np.uint16) + np.uint16(1)).view(np.float16), s)
    s = np.where(flat, np.float32(1), s.astype(np.float32))
    r = lo / s
    step = np.ldexp(np.float32(1), np.frexp(np.abs(r) + np.float32(16))[1] - 11).astype(np.float32)
    r = np.rint(r / step) * step
    n = np.clip(np.rint((f - s * r) / s), 0, 15)
    n = np.where(flat | bad, 0, n).astype(np.uint8)
    s, r = np.where(flat, lo, s), np.where(flat, np.float32(1), r)
    p = np.concatenate([s, r], -1).astype(np.float16)
    p = np.where(bad, np.array([NAN_ROW], np.uint16).view(np.float16), p)
    return n, p


def values(n, p):
    """What codes and (s, r) stand for, in 64 bits."""
    p = p.astype(np.float64)
    return p[..., :1] * (n + p[..., 1:])


def pack(kn, kp, vn, vp):
    """Pages [..., 16 (D + 8)] of codes [..., 16, D] and (s, r) [..., 16, 2]."""
    def flat(a):
        return np.ascontiguousarray(a).view(np.uint8).reshape(a.shape[:-2] + (-1,))
    codes = [n[..., 0::2] | (n[..., 1::2] << 4) for n in (kn, vn)]
    return np.concatenate([flat(codes[0]), flat(codes[1]), flat(kp), flat(vp)], -1)


def unpack(pages, d):
    """pack's inverse: (kn, kp, vn, vp)."""
    lead = pages.shape[:-1]
    out = []
    for i in range(2):
        c = pages[..., i * 8 * d:(i + 1) * 8 * d].reshape(lead + (PAGE, d // 2))
        n = np.stack([c & 15, c >> 4], -1).reshape(lead + (PAGE, d))
        at = 16 * d + 64 * i
        p = np.ascontiguousarray(pages[..., at:at + 64]).view(np.float16).reshape(lead + (PAGE, 2))
        out += [n, p]
    return out[0], out[1], out[2], out[3]


class Q4Cache:
    """K and V of `lens` tokens per sequence in 4-bit pages, and what they stand for
    on the host as [B][Hkv][T][D]; slots outside the sequences hold NaN rows."""

    def __init__(self, rng, lens, hkv, d, scale=1.0, offset=0.0, cap=None, slack=3):
        self.lens = np.asarray(lens, np.int32)
        self.hkv, self.d = hkv, d
        B, T = len(self.lens), max(1, int(self.lens.max()))
        self.cap = T if cap is None else cap
        self.bt, self.pages = make_block_tables(rng, self.lens, slack_pages=slack)
        rows = (hkv, self.pages, PAGE, d)
        kv = [(rng.standard_normal(rows) * scale + offset).astype(np.float16) for _ in range(2)]
        kn, kp = quantise(kv[0])
        vn, vp = quantise(kv[1])
        self.parts = [kn, kp, vn, vp]
        used = np.zeros((self.pages, PAGE), bool)
        for b, n in enumerate(self.lens):
            j = np.arange(int(n))
            used[self.bt[b, j // PAGE], j % PAGE] = True
        for i in (1, 3):
            self.parts[i][:, ~used] = np.nan
        self.T, self.B = T, B
        self.stand()

    def stand(self):
        """Host values of the sequences' slots from the present parts."""
        kn, kp, vn, vp = self.parts
        self.k = np.zeros((self.B, self.hkv, self.T, self.d))
        self.v = np.zeros_like(self.k)
        with np.errstate(invalid="ignore"):
            kx, vx = values(kn, kp), values(vn, vp)
        for b, n in enumerate(self.lens):
            j = np.arange(int(n))
            self.k[b, :, :n] = kx[:, self.bt[b, j // PAGE], j % PAGE]
            self.v[b, :, :n] = vx[:, self.bt[b, j // PAGE], j % PAGE]

    def upload(self):
        self.pool = to_gpu(pack(*self.parts))
        self.bt_d, self.lens_d = to_gpu(self.bt), to_gpu(self.lens)
        return self


def rotated(x, pos, theta):
    """x [..., D] at position pos (broadcast over [...]) in 64 bits, and the bound on
    what the fp32 products and sums before the one rounding to fp16 add."""
    x = x.astype(np.float64)
    h = x.shape[-1] // 2
    if theta == 0:
        return x, np.zeros_like(x)
    ang = np.asarray(pos, np.float64)[..., None] * theta ** (-np.arange(h) / h)
    c, s = np.cos(ang), np.sin(ang)
    a, b = x[..., :h], x[..., h:]
    y = np.concatenate([a * c - b * s, b * c + a * s], -1)
    # sine, cosine, product and sum are rounded to fp32 once each; the angle of 2^31 turns
    # to 2^-53 of its size in either computation
    size = np.abs(a) + np.abs(b)
    e = 4 * U32 * size + 4 * 2.0 ** -52 * np.abs(ang) * size
    return y, np.concatenate([e, e], -1)
