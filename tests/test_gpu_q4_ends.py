"""4-bit rows that reach fp16's largest value: a row's ends may stand for a little more
than 65504 (s and r are rounded), which is read back and attended as 65504, never as
infinity (tolerances: bounded_util, q4_util)."""
import numpy as np
import pytest

import kvhp
from bounded_util import attend, check
from gpu_util import from_gpu, note, sync
from q4_util import Q4Cache, quantise, values
from test_gpu_q4 import _decode, _prefill, _q

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

MOST = 65504.0
KINDS = {"0 to the largest": (0, MOST), "the least to 0": (-MOST, 0), "both ends": (-MOST, MOST),
         "the largest and near it": (MOST - 512, MOST), "the least and near it": (-MOST, -MOST + 1024),
         "one end near": (-65408, 32000)}


def _cache(rng, kind, n, d):
    """n keys whose V rows all hold the two values of `kind`, in an order of their own."""
    c = Q4Cache(rng, [n], 2, d)
    x = rng.permuted(np.tile(np.array(KINDS[kind], np.float16), (2, 1, 1, d // 2)), axis=-1)
    vn, vp = quantise(np.broadcast_to(x, c.parts[2].shape))
    c.parts[2], c.parts[3] = vn, np.where(np.isnan(c.parts[3]), c.parts[3], vp)
    c.stand()
    return c.upload()


def test_rows_stand_for_more():
    """What the cases are about, on the host: ends past 65520 but for the last kinds."""
    past = 0
    for lo, hi in KINDS.values():
        n, p = quantise(np.array([lo, hi] * 4, np.float16))
        past += np.abs(values(n, p)).max() >= 65520
    assert past >= 3


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [40, 64, 128])
def test_gather_at_the_ends(kind, d):
    c = _cache(np.random.default_rng(d), kind, 37, d)
    k, v = (torch.empty((1, 2, 37, d), dtype=torch.float16, device="cuda") for _ in range(2))
    note(f"q4_gather {kind} d={d}")
    kvhp.q4_gather(c.pool, c.bt_d, c.lens_d, k, v)
    sync()
    assert np.array_equal(from_gpu(v), np.clip(c.v, -MOST, MOST).astype(np.float16))
    assert np.array_equal(from_gpu(k), c.k.astype(np.float16))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("n", [1, 150, 5000])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_attention_at_the_ends(kind, n, d):
    """Every weighted mean of such rows, in one piece and joined from several."""
    rng = np.random.default_rng(n + d)
    c = _cache(rng, kind, n, d)

    def holds(got, q, keys, what):
        for h in range(2):
            hs = slice(4 * h, 4 * h + 4)
            o, tol, _, _, _ = attend(q[hs], c.k[0, h, :keys], c.v[0, h, :keys], np.ones(keys, bool))
            assert np.isfinite(got[hs]).all(), f"{what} head {h}"
            check(got[hs], np.clip(o, -MOST, MOST), tol, f"{what} head {h}")

    q = _q(rng, 1, 8, d)
    note(f"q4_decode {kind} n={n} d={d}")
    holds(_decode(q, c)[0], q[0], n, "decode")
    for R in (1, 40, 150):
        if R > n:
            continue
        q = _q(rng, 1, R, 8, d)
        note(f"q4_prefill {kind} n={n} d={d} rows={R}")
        got, _ = _prefill(q, c, [n - R])
        for r in range(0, R, 13):
            holds(got[0, r], q[0, r], n - R + r + 1, f"row {r} of {R}")
