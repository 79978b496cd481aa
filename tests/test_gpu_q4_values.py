"""Attention over 4-bit caches whose rows are of all sizes up to fp16's largest, at row
counts on both sides of where one kernel hands over to another (tolerances:
bounded_util, q4_util)."""
import numpy as np
import pytest

import kvhp
from bounded_util import PAGE
from gpu_util import note
from q4_util import Q4Cache, quantise
from test_gpu_q4 import _check_decode, _check_prefill, _prefill, _q

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROWS = [5, 40, 150]   # 20, 160 and 600 (row, query head) pairs of a KV head


def _by_prompt_kernel(c, rows, hq):
    """Whether the calls of q4_prefill at head_dim 64 or 128 run on the kernel that works on 128
    pairs a workgroup, by what the size query says: that one keeps a number beside its ranges'
    partials, the other, 16 pairs a wave, cuts every context of more than a tile that these
    tests have into ranges."""
    n = kvhp.q4_prefill_workspace_bytes(c.B, rows, hq, c.hkv, c.d, c.cap)
    partials = 4 * c.B * rows * hq * (c.d + 2)
    assert n % partials in (0, 4)
    return n == 0 or n % partials == 4


def _rows_on_both_sides(c, hq):
    if c.d in (64, 128):
        assert [_by_prompt_kernel(c, R, hq) for R in ROWS] == [False, True, True]
    return ROWS


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
    for c.cap in (256, n):   # a limit of four tiles, from which on few rows have a kernel of their own
        for R in ROWS if c.cap == n else _rows_on_both_sides(c, 8):
            note(f"q4 equal values {value} d={d} rows={R} cap={c.cap}")
            got, _ = _check_prefill(q[R], c, [n - R], f"{R} rows", every=3)
            assert np.isfinite(got).all()
    if d != 96:   # there a tile's largest scale has a say in where small weights end
        before = keys[0] - (n - most)
        assert np.array_equal(got[0, :before], clean[0, :before])
    note(f"q4_decode equal values {value} d={d}")
    _check_decode(q[5][:, -1], c)


@pytest.mark.parametrize("scale,offset", [(1e-3, 0.0), (30.0, 0.0), (1.0, 40.0), (3e-6, 0.0), (0.01, -3.0),
                                          (200.0, 5000.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_many_sizes(scale, offset, d):
    """Tiny, large and offset keys and values under a step's rows, a chunk's and a prompt's."""
    rng = np.random.default_rng(int(100 * scale) + d)
    c = Q4Cache(rng, [300, 187], 2, d, scale=scale, offset=offset).upload()
    for R in _rows_on_both_sides(c, 8):
        # large keys sharpen the softmax, so that few keys count; small ones level it
        q = (_q(rng, 2, R, 8, d) * np.float16(1 / max(scale, 1))).astype(np.float16)
        note(f"q4_prefill rows={R} scale={scale} offset={offset} d={d}")
        _check_prefill(q, c, [300 - R, 187 - R], f"{R} rows", every=19)


@pytest.mark.parametrize("equal", [300.0, 33000.0, -65504.0])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_mixed_sizes(d, equal):
    """Rows whose scales differ by many orders of magnitude side by side, rows of equal
    values and rows at both of fp16's ends among them."""
    rng = np.random.default_rng(d)
    c = Q4Cache(rng, [330, 190], 2, d)
    for i in (0, 2):
        x = rng.standard_normal((2, c.pages, PAGE, d))
        size = 10.0 ** rng.uniform(-6, 2, (2, c.pages, PAGE, 1))
        if i == 0:
            size = np.minimum(size, 3.0)      # scores that an exponential can tell apart
        x = x * size
        x[:, :, 3] = x[:, :, 3, :1]           # equal values
        if i == 2:
            x[:, :, 5] = equal
            x[:, :, 7] = np.where(x[:, :, 7] > 0, 65504, -65504)
            x[:, :, 8] = 0
        n, p = quantise(x.astype(np.float16))
        old = c.parts[i + 1]
        c.parts[i], c.parts[i + 1] = n, np.where(np.isnan(old), old, p)
    c.stand()
    c.upload()
    for R in _rows_on_both_sides(c, 8):
        note(f"q4 mixed rows={R} equal={equal} d={d}")
        q = _q(rng, 2, R, 8, d)
        _check_prefill(q, c, [330 - R, 190 - R], f"{R} rows", every=19)
    _check_decode(q[:, -1], c)


@pytest.mark.parametrize("n,rows", [(5000, 17), (5000, 40), (8191, 33), (3001, 129)])
@pytest.mark.parametrize("d", [64, 128])
def test_ranges_of_a_long_cache(n, rows, d):
    """A chunk's rows over ranges of keys, on the kernel of 128 pairs."""
    rng = np.random.default_rng(n + rows + d)
    c = Q4Cache(rng, [n], 2, d).upload()
    assert _by_prompt_kernel(c, rows, 8) and kvhp.q4_prefill_workspace_bytes(1, rows, 8, 2, d, n) > 0
    note(f"q4_prefill {rows} rows behind {n} keys, d={d}")
    _check_prefill(_q(rng, 1, rows, 8, d), c, [n - rows], every=16)
    _check_prefill(_q(rng, 1, rows, 8, d), c, [17], every=16)
