"""Attention over 4-bit caches whose rows are of all sizes up to fp16's largest, at row
counts on both sides of where one kernel hands over to another (tolerances:
bounded_util, q4_util)."""
import numpy as np
import pytest

from bounded_util import PAGE, attend, check
from gpu_util import note
from q4_util import Q4Cache, quantise
from test_gpu_q4 import _check_decode, _check_prefill, _prefill, _q

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROWS = [5, 40, 150]   # 20, 160 and 600 (row, query head) pairs of a KV head


def _put(c, i, b, key, rows):
    """Rows fp16 [Hkv][D] as sequence b's K (i = 0) or V (2) of `key`."""
    n, p = quantise(np.asarray(rows, np.float16))
    page, at = c.bt[b, key // PAGE], key % PAGE
    c.parts[i][:, page, at], c.parts[i + 1][:, page, at] = n, p


@pytest.mark.parametrize("value", [20000, 32752, 32768, -32768, 40000, -40000, 65504, -65504])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_equal_values_up_to_the_largest(value, d):
    """V rows of one large value each: rows that see them get their share, rows before them
    none of it."""
    rng = np.random.default_rng(abs(value) + d)
    n, keys = 170, (70, 127, 160)
    c = Q4Cache(rng, [n], 2, d).upload()
    q = {R: _q(rng, 1, R, 8, d) for R in ROWS}
    most = ROWS[-1]
    note(f"q4 equal values d={d}: without")
    clean = _prefill(q[most], c, [n - most])[0]
    for k in keys:
        _put(c, 2, 0, k, np.full((2, d), value))
    c.stand()
    c.upload()
    for R in ROWS:
        note(f"q4 equal values {value} d={d} rows={R}")
        got, _ = _check_prefill(q[R], c, [n - R], f"{R} rows", every=3)
        assert np.isfinite(got).all()
    if d != 96:   # there a tile's largest scale has a say in where small weights end
        before = keys[0] - (n - most)
        assert np.array_equal(got[0, :before], clean[0, :before])
    note(f"q4_decode equal values {value} d={d}")
    _check_decode(q[5][:, -1], c)
