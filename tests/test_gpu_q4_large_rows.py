"""Small weights beside V rows of very large values that next to nothing is attended of: a
key's weight is as exact as if those rows were any others."""
import numpy as np
import pytest

from bounded_util import attend, check
from gpu_util import note
from q4_util import PAGE, Q4Cache, quantise
from test_gpu_q4 import _decode, _prefill

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

LARGE = {"equal": lambda rng, d: np.full(d, 65504.0), "minus": lambda rng, d: np.full(d, -33000.0),
         "both": lambda rng, d: rng.choice([-65504.0, 65504.0], d), "some": lambda rng, d: 300 * rng.standard_normal(d)}


def _cache(rng, n, hkv, d, kind, batch=1):
    """n keys that `batch` sequences share: the first has twice as much weight as all others,
    which weigh the same; in every tile of 64 one has almost none, and its V is large.  All
    other V rows hold the same values of 0.05 .. 0.15 in orders of their own, so that their
    weights' roundings do not cancel."""
    c = Q4Cache(rng, [n], hkv, d)
    shape = c.parts[0].shape
    x = rng.permuted(np.broadcast_to(np.linspace(0.05, 0.15, d), shape), axis=-1)
    k = np.zeros(shape)
    j = np.arange(n)
    page, at = c.bt[0, j // PAGE], j % PAGE
    k[:, page[0], at[0]] = np.log(2.0 * n)     # equal values: keys stand for them exactly
    for i in range(1 + rng.integers(0, 60), n, 64):
        k[:, page[i], at[i]] = -30
        x[:, page[i], at[i]] = LARGE[kind](rng, d)
    for i, rows in ((0, k), (2, x)):
        codes, p = quantise(rows.astype(np.float16))
        c.parts[i], c.parts[i + 1] = codes, np.where(np.isnan(c.parts[i + 1]), c.parts[i + 1], p)
    c.stand()
    c.lens, c.bt = np.repeat(c.lens, batch), np.repeat(c.bt, batch, 0)
    return c.upload()


def _holds(got, q, c, h, keys, what):
    """The tolerance of `attend`, whose absolute part goes by the largest |V|: here by the
    largest of the rows that weigh.  The large ones' weights are 2^-43 of their neighbours',
    and are rounded to 2^-11 of themselves or lost."""
    k, v = c.k[0, h, :keys], c.v[0, h, :keys]
    o, tol, _, _, _ = attend(q, k, v, np.ones(keys, bool))
    s = q.astype(np.float64) @ k.T / np.sqrt(c.d)
    l = np.exp(s - s.max(1, keepdims=True)).sum(1, keepdims=True)
    tol = tol - keys * 2.0 ** -25 * (np.abs(v).max() - 0.16) / l + (keys // 64 + 1) * 2.0 ** -43 * np.abs(v).max()
    check(got, o, tol, what)


def _q(rng, d, *lead):
    """q.k / sqrt(d) is a key's one value, but for a few per cent that differ by head."""
    q = np.full(lead + (d,), 1 / np.sqrt(d)) * rng.uniform(0.98, 1.02, lead + (1,))
    return q.astype(np.float16)


@pytest.mark.parametrize("kind", list(LARGE))
@pytest.mark.parametrize("G,d", [(1, 64), (5, 64), (9, 64), (4, 128), (8, 128), (9, 128), (1, 96), (2, 256)])
def test_decode_beside_large_rows(G, d, kind):
    """So many sequences and heads that a wave takes 16 tiles, the first key's among them."""
    rng = np.random.default_rng(G + d)
    hkv, B = 64, 24 if d in (64, 128) else 64
    c = _cache(rng, 1000, hkv, d, kind, B)
    q = _q(rng, d, B, G * hkv)
    for c.cap in (4096, 1000):   # splits by the batch; one of eight waves
        note(f"q4_decode {B} sequences {G * hkv}/{hkv} x {d} cap={c.cap} beside {kind}")
        got = _decode(q, c)
        for b in (0, B // 2, B - 1):
            for h in (0, 1, 30, hkv - 1):
                hs = slice(G * h, G * (h + 1))
                _holds(got[b, hs], q[b, hs], c, h, 1000, f"sequence {b} head {h}")


@pytest.mark.parametrize("kind", list(LARGE))
@pytest.mark.parametrize("rows", [3, 20, 70])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_rows_beside_large_rows(d, rows, kind):
    rng = np.random.default_rng(rows + d)
    for n in (700, 5000):
        c = _cache(rng, n, 2, d, kind)
        q = _q(rng, d, 1, rows, 8)
        note(f"q4_prefill {rows} rows behind {n} keys x {d} beside {kind}")
        got, _ = _prefill(q, c, [n - rows])
        for r in {0, rows // 2, rows - 1}:
            for h in range(2):
                hs = slice(4 * h, 4 * h + 4)
                _holds(got[0, r, hs], q[0, r, hs], c, h, n - rows + r + 1, f"row {r} of {rows}, {n} keys, head {h}")
