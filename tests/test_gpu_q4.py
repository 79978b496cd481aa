"""Attention over a cache held in 4 bits, against its definition in 64 bits
(tolerances: bounded_util, q4_util)."""
import numpy as np
import pytest

import kvhp
from bounded_util import PAGE, U16, U32, attend, check, workspace
from gpu_util import from_gpu, note, sync, to_gpu
from q4_util import Q4Cache, values

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HEADS = [(32, 8, 128), (32, 4, 64), (14, 2, 64), (32, 8, 64), (4, 4, 128), (1, 1, 64), (20, 1, 128),
         (34, 2, 64)]
ODD = [(8, 2, 96), (5, 1, 256), (6, 2, 8), (4, 4, 40)]   # the kernel for any shape


def _q(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def _decode(q, c, stream=None):
    hq, d = q.shape[1:]
    ws = workspace(kvhp.q4_decode_workspace_bytes(len(c.lens), hq, c.hkv, d, c.cap))
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    kvhp.q4_decode(to_gpu(q), c.pool, c.bt_d, c.lens_d, out, hq, c.hkv, d, c.cap, workspace=ws,
                   stream=stream)
    sync()
    return from_gpu(out)


def _check_decode(q, c, what=""):
    got = _decode(q, c)
    G = q.shape[1] // c.hkv
    for b in range(len(c.lens)):
        n = min(int(c.lens[b]), c.cap)
        if n <= 0:
            assert (got[b] == 0).all()
            continue
        for h in range(c.hkv):
            hs = slice(h * G, (h + 1) * G)
            o, tol, _, _, _ = attend(q[b, hs], c.k[b, h, :n], c.v[b, h, :n], np.ones(n, bool))
            check(got[b, hs], o, tol, f"{what} sequence {b} head {h}")
    return got


@pytest.mark.parametrize("hq,hkv,d", HEADS + ODD)
def test_decode_heads(hq, hkv, d):
    rng = np.random.default_rng(hq + d)
    c = Q4Cache(rng, [133, 64, 1, 0, 300], hkv, d).upload()
    note(f"q4_decode {hq}/{hkv} x {d}")
    _check_decode(_q(rng, 5, hq, d), c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 511, 513, 700,
                               1023, 1025, 1500, 2049, 3001, 4097])
def test_decode_lengths(n, d):
    rng = np.random.default_rng(n + d)
    c = Q4Cache(rng, [n], 2, d).upload()
    note(f"q4_decode n={n} d={d}")
    _check_decode(_q(rng, 1, 8, d), c)


@pytest.mark.parametrize("B", [2, 7, 16, 24, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_batches(B, d):
    """Ragged batches, sequences without keys among them, and more room than they need."""
    rng = np.random.default_rng(B + d)
    lens = rng.integers(0, 1400, B)
    lens[0], lens[-1] = 0, 1400
    c = Q4Cache(rng, lens, 2, d).upload()
    note(f"q4_decode B={B} d={d}")
    q = _q(rng, B, 8, d)
    _check_decode(q, c)
    for cap in (3000, 333):     # a limit above and below the lengths
        c.cap = cap
        _check_decode(q, c, f"cap {cap}")


@pytest.mark.parametrize("scale,offset", [(1e-3, 0.0), (30.0, 0.0), (1.0, 40.0), (3e-6, 0.0), (0.01, -3.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_values_of_many_sizes(scale, offset, d):
    rng = np.random.default_rng(int(100 * scale) + d)
    c = Q4Cache(rng, [200, 77], 2, d, scale=scale, offset=offset).upload()
    # keys of size 30 sharpen the softmax, so that few keys count; small ones level it
    q = (_q(rng, 2, 8, d) * np.float16(1 / max(scale, 1))).astype(np.float16)
    note(f"q4 values scale={scale} offset={offset} d={d}")
    _check_decode(q, c)
    _check_prefill(np.repeat(q[:, None], 5, 1), c, [195, 72], "prefill")


@pytest.mark.parametrize("d", [64, 128])
def test_mixed_rows(d):
    """Rows whose scales differ by many orders of magnitude side by side, flat rows and rows
    at fp16's limits among them."""
    rng = np.random.default_rng(d)
    c = Q4Cache(rng, [330, 90], 2, d)
    from q4_util import quantise
    for i in (0, 2):
        x = rng.standard_normal((2, c.pages, PAGE, d))
        size = 10.0 ** rng.uniform(-6, 2, (2, c.pages, PAGE, 1))
        if i == 0:
            size = np.minimum(size, 3.0)      # scores that an exponential can tell apart
        x = x * size
        x[:, :, 3] = x[:, :, 3, :1]           # equal values
        if i == 2:
            x[:, :, 7] = np.where(x[:, :, 7] > 0, 65504, -65504)
            x[:, :, 8] = 0
        n, p = quantise(x.astype(np.float16))
        old = c.parts[i + 1]
        c.parts[i], c.parts[i + 1] = n, np.where(np.isnan(old), old, p)
    c.stand()
    c.upload()
    note(f"q4 mixed rows d={d}")
    q = _q(rng, 2, 8, d)
    _check_decode(q, c)
    _check_prefill(np.repeat(q[:, None], 5, 1), c, [200, 85], "prefill")


def _prefill(q, c, start, lse=True, stream=None, lens=True):
    B, R, hq, d = q.shape
    ws = workspace(kvhp.q4_prefill_workspace_bytes(B, R, hq, c.hkv, d, c.cap))
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    ls = torch.full((B, hq, R), 7.0, device="cuda") if lse else None
    kvhp.q4_prefill(to_gpu(q), c.pool, c.bt_d, out, hq, c.hkv, d, c.cap,
                    q_start=None if start is None else to_gpu(np.asarray(start, np.int32)),
                    seq_lens=c.lens_d if lens else None, lse=ls, workspace=ws, stream=stream)
    sync()
    return from_gpu(out), None if ls is None else from_gpu(ls)


def _check_prefill(q, c, start, what="", lens=True, every=1):
    """Every `every`-th row, and the padding rows."""
    got, ls = _prefill(q, c, start, lens=lens)
    B, R, hq, d = q.shape
    G = hq // c.hkv
    for b in range(B):
        n = min(int(c.lens[b]) if lens else c.cap, c.cap)
        first = 0 if start is None else int(start[b])
        for r in range(R):
            p = first + r
            if p < 0 or p >= n:
                assert (got[b, r] == 7).all() and (ls[b, :, r] == 7).all(), f"{what} padding {b}, {r}"
                continue
            if r % every and r != R - 1:
                continue
            for h in range(c.hkv):
                hs = slice(h * G, (h + 1) * G)
                k, v = c.k[b, h, :p + 1], c.v[b, h, :p + 1]
                o, tol, _, l, ds = attend(q[b, r, hs], k, v, np.ones(p + 1, bool))
                check(got[b, r, hs], o, tol, f"{what} sequence {b} row {r} head {h}")
                check(ls[b, hs, r], l, ds + (p + 8) * U32 + 4 * U32 * np.abs(l), f"{what} lse {b} {r} {h}")
    return got, ls


@pytest.mark.parametrize("hq,hkv,d", HEADS + ODD)
def test_prefill_heads(hq, hkv, d):
    rng = np.random.default_rng(hq + d + 1)
    c = Q4Cache(rng, [37, 90, 0], hkv, d).upload()
    note(f"q4_prefill {hq}/{hkv} x {d}")
    _check_prefill(_q(rng, 3, 90, hq, d), c, None, every=7)
    c = Q4Cache(rng, [37, 140], hkv, d).upload()
    _check_prefill(_q(rng, 2, 9, hq, d), c, [28, 131])


@pytest.mark.parametrize("rows", [1, 2, 7, 16, 33, 128, 129])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_chunks(rows, d):
    """Chunks behind cached keys, left and right padding, sequences of other lengths."""
    rng = np.random.default_rng(rows + d)
    lens = [rows + 300, rows + 11, rows, max(1, rows - 1), rows + 64]
    c = Q4Cache(rng, lens, 2, d).upload()
    note(f"q4_prefill chunk rows={rows} d={d}")
    q = _q(rng, 5, rows, 8, d)
    _check_prefill(q, c, [n - rows for n in lens], every=3)
    _check_prefill(q, c, [0, 5, -3, rows, 63], every=5)
    _check_prefill(q, c, [-rows, 1 << 30, -(1 << 31), (1 << 31) - 1, 64], every=5)


@pytest.mark.parametrize("S,heads", [(64, (8, 2, 64)), (65, (8, 2, 128)), (200, (14, 2, 64)),
                                     (777, (7, 1, 64)), (513, (4, 1, 128)), (1024, (2, 2, 64))])
def test_prefill_prompts(S, heads):
    hq, hkv, d = heads
    rng = np.random.default_rng(S)
    c = Q4Cache(rng, [S, max(1, S // 3)], hkv, d).upload()
    note(f"q4_prefill prompt S={S} {heads}")
    _check_prefill(_q(rng, 2, S, hq, d), c, None, every=37)


@pytest.mark.parametrize("n,rows", [(5000, 1), (5000, 9), (3001, 40), (8191, 5)])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_few_rows_long_cache(n, rows, d):
    rng = np.random.default_rng(n + rows + d)
    c = Q4Cache(rng, [n], 2, d).upload()
    note(f"q4_prefill {rows} rows behind {n} keys, d={d}")
    _check_prefill(_q(rng, 1, rows, 8, d), c, [n - rows], every=4)
    _check_prefill(_q(rng, 1, rows, 8, d), c, [17], every=4)


def test_prefill_without_lengths_and_lse():
    rng = np.random.default_rng(5)
    c = Q4Cache(rng, [160, 160], 2, 64).upload()
    q = _q(rng, 2, 50, 8, 64)
    note("q4_prefill without lengths")
    a, _ = _check_prefill(q, c, [110, 20], lens=False)
    b, ls = _prefill(q, c, [110, 20], lse=False, lens=False)
    assert ls is None and np.array_equal(a, b)


@pytest.mark.parametrize("d", [64, 128, 40])
def test_hidden_rows_reach_nothing(d):
    """NaN rows behind the lengths (Q4Cache puts them there), in slots that a row does not
    see yet, in pages that no table names; a row that sees one is NaN, the others as if it
    were any other."""
    rng = np.random.default_rng(d)
    c = Q4Cache(rng, [150, 71], 2, d).upload()
    q = _q(rng, 2, 150, 8, d)
    note(f"q4_prefill NaN rows d={d}")
    clean, lc = _prefill(q, c, None)
    for which in (1, 3):                    # K's numbers, V's
        for key in (0, 40, 63, 64, 100, 149):
            old = c.parts[which].copy()
            c.parts[which][1, c.bt[0, key // PAGE], key % PAGE] = np.nan
            c.upload()
            note(f"q4_prefill NaN part {which} key {key} d={d}")
            got, ls = _prefill(q, c, None)
            assert np.array_equal(got[1], clean[1]) and np.array_equal(got[0, :, :4], clean[0, :, :4])
            assert np.array_equal(got[0, :key], clean[0, :key])
            assert np.isnan(got[0, key:, 4:].astype(np.float32)).all()
            want = np.isnan(ls[0, 4:, key:]) if which == 1 else ls[0, 4:, key:] == lc[0, 4:, key:]
            assert want.all() and np.array_equal(ls[0, :, :key], lc[0, :, :key])
            c.parts[which] = old
    c.upload()
    note(f"q4_decode NaN rows d={d}")
    clean = _decode(q[:, -1], c)
    for which in (1, 3):
        old = c.parts[which].copy()
        c.parts[which][0, c.bt[1, 70 // PAGE], 70 % PAGE] = np.nan
        c.upload()
        got = _decode(q[:, -1], c)
        assert np.isnan(got[1, :4].astype(np.float32)).all()
        assert np.array_equal(got[0], clean[0]) and np.array_equal(got[1, 4:], clean[1, 4:])
        c.lens_d = to_gpu(np.array([150, 70], np.int32))   # hidden now
        assert np.isfinite(_decode(q[:, -1], c).astype(np.float32)).all()
        c.parts[which] = old
        c.upload()


def test_garbage_in_hidden_slots():
    """Any bytes behind the lengths and in other pages: the same bits."""
    rng = np.random.default_rng(3)
    for d in (64, 128, 96):
        c = Q4Cache(rng, [75, 33, 1], 2, d).upload()
        q = _q(rng, 3, 8, d)
        qp = _q(rng, 3, 33, 8, d)
        note(f"q4 garbage d={d}")
        a, (b, bl) = _decode(q, c), _prefill(qp, c, [42, 0, 0])
        used = np.zeros((c.pages, PAGE), bool)
        for i, n in enumerate(c.lens):
            j = np.arange(int(n))
            used[c.bt[i, j // PAGE], j % PAGE] = True
        for k in range(4):
            junk = np.frombuffer(rng.bytes(c.parts[k].nbytes), c.parts[k].dtype).reshape(c.parts[k].shape)
            if k % 2 == 0:
                junk = junk & 15
            c.parts[k] = np.where(used[None, :, :, None], c.parts[k], junk)
        c.upload()
        assert np.array_equal(_decode(q, c), a)
        got = _prefill(qp, c, [42, 0, 0])
        assert np.array_equal(got[0], b) and np.array_equal(got[1], bl)


def test_page_ids_are_clamped_for_reads():
    """-1 and ids past the pool read the pool's first and last page."""
    rng = np.random.default_rng(8)
    c = Q4Cache(rng, [200], 2, 64)
    for i in (1, 3):
        c.parts[i] = np.where(np.isnan(c.parts[i]), np.float16(0.25), c.parts[i])
    same = c.bt.copy()
    same[0, 2], same[0, 5] = 0, c.pages - 1
    c.bt = same
    c.stand()
    c.upload()
    q = _q(rng, 1, 8, 64)
    a, b = _check_decode(q, c), _prefill(q[:, None], c, [199])
    bad = same.copy()
    bad[0, 2], bad[0, 5] = -1, 1 << 30
    c.bt_d = to_gpu(bad)
    note("q4 page ids outside the pool")
    assert np.array_equal(_decode(q, c), a)
    assert np.array_equal(_prefill(q[:, None], c, [199])[0], b[0])


def test_shared_pages():
    """Two sequences over the same prefix pages."""
    rng = np.random.default_rng(12)
    c = Q4Cache(rng, [160, 170], 2, 64)
    c.bt[1, :6] = c.bt[0, :6]
    c.stand()
    c.upload()
    note("q4 shared pages")
    _check_decode(_q(rng, 2, 8, 64), c)
    _check_prefill(_q(rng, 2, 20, 8, 64), c, [140, 150])


def test_rows_equal_decode():
    """One row of q4_prefill is q4_decode's output within both tolerances."""
    rng = np.random.default_rng(2)
    c = Q4Cache(rng, [333, 1000], 2, 128).upload()
    q = _q(rng, 2, 8, 128)
    note("q4_prefill of one row against q4_decode")
    _check_decode(q, c)
    _check_prefill(q[:, None], c, [332, 999])


def _together(c, q, k, v, pos, bufs):
    """A step: append the token's K and V, attend; and a chunk of the last rows."""
    qo, out, po, ls, dws, pws = bufs
    kvhp.q4_rope_append(q, k, v, pos, qo, c.pool, c.bt_d, 8, 2, 64, 10000.0)
    kvhp.q4_decode(qo[:, 0], c.pool, c.bt_d, c.lens_d, out, 8, 2, 64, c.cap, workspace=dws)
    kvhp.q4_prefill(qo, c.pool, c.bt_d, po, 8, 2, 64, c.cap, q_start=pos, seq_lens=c.lens_d, lse=ls,
                    workspace=pws)


def test_steps_on_streams_and_in_graphs():
    """Append and attention as a serving step makes them: eager, on another stream and
    replayed from a graph with eager work between, bit for bit."""
    rng = np.random.default_rng(21)
    lens = [900, 77, 1200, 16]
    c = Q4Cache(rng, lens, 2, 64).upload()
    start = c.pool.clone()
    pos = to_gpu(np.asarray(lens, np.int32) - 1)
    q, k, v = (to_gpu(_q(rng, 4, 1, h, 64)) for h in (8, 2, 2))

    def buffers():
        n = kvhp.q4_decode_workspace_bytes(4, 8, 2, 64, c.cap)
        m = kvhp.q4_prefill_workspace_bytes(4, 1, 8, 2, 64, c.cap)
        return (torch.zeros_like(q), torch.zeros_like(q[:, 0]), torch.zeros_like(q),
                torch.zeros((4, 8, 1), device="cuda"), workspace(n), workspace(m))

    note("q4 step: eager")
    want = buffers()
    _together(c, q, k, v, pos, want)
    sync()
    pool = c.pool.clone()
    assert not torch.equal(pool, start)
    # both tolerances, where a weighted mean of |V| is below 2
    check(from_gpu(want[1]).astype(np.float64), from_gpu(want[2])[:, 0].astype(np.float64),
          4 * U16 * np.abs(from_gpu(want[1])).astype(np.float64) + 8 * U16)
    note("q4 step: another stream")
    c.pool.copy_(start)
    got = buffers()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _together(c, q, k, v, pos, got)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want[:4], got[:4])) and torch.equal(c.pool, pool)
    graph = torch.cuda.CUDAGraph()
    got = buffers()
    with torch.cuda.graph(graph):
        _together(c, q, k, v, pos, got)
    src = k.clone()
    for i in range(4):
        note(f"q4 step: replay {i}")
        k.copy_(src * (1 + i))
        c.pool.copy_(start)
        for t in got[:4]:
            t.fill_(9)
        for t in got[4:]:
            if t is not None:
                t.fill_(255)
        graph.replay()
        sync()
        replayed = [t.clone() for t in got[:4]] + [c.pool.clone()]
        c.pool.copy_(start)
        eager = buffers()
        _together(c, q, k, v, pos, eager)
        sync()
        assert all(torch.equal(a, b) for a, b in zip(replayed, list(eager[:4]) + [c.pool]))


def test_repeated_calls_are_the_same_bits():
    rng = np.random.default_rng(31)
    c = Q4Cache(rng, [2000, 900, 1999], 2, 128).upload()
    q = _q(rng, 3, 8, 128)
    a = _decode(q, c)
    qp = _q(rng, 3, 70, 8, 128)
    b = _prefill(qp, c, [1900, 800, 1000])
    for i in range(5):
        note(f"q4 repeat {i}")
        assert np.array_equal(_decode(q, c), a)
        got = _prefill(qp, c, [1900, 800, 1000])
        assert np.array_equal(got[0], b[0]) and np.array_equal(got[1], b[1])


def test_serving_from_four_bits():
    """A prompt appended in two chunks, then tokens one by one: each attention is that over
    what the cache holds, read back by q4_gather."""
    rng = np.random.default_rng(4)
    hq, hkv, d, S, steps = 8, 2, 64, 90, 5
    T = S + steps
    x = to_gpu(_q(rng, 1, T, hq + 2 * hkv, d))
    pages = (T + PAGE - 1) // PAGE
    bt = to_gpu(rng.permutation(pages).astype(np.int32)[None])
    pool = torch.zeros((hkv, pages, kvhp.q4_page_bytes(d)), dtype=torch.uint8, device="cuda")
    outs, qs = [], []
    at = 0
    for R in [50, 40] + [1] * steps:
        note(f"q4 serving: {R} rows at {at}")
        rows = x[:, at:at + R]
        pos = torch.tensor([at], dtype=torch.int32, device="cuda")
        lens = torch.tensor([at + R], dtype=torch.int32, device="cuda")
        q = torch.empty((1, R, hq, d), dtype=torch.float16, device="cuda")
        kvhp.q4_rope_append(rows[:, :, :hq], rows[:, :, hq:hq + hkv], rows[:, :, hq + hkv:], pos, q,
                            pool, bt, hq, hkv, d, 10000.0)
        out = torch.empty_like(q)
        if R == 1:
            kvhp.q4_decode(q[:, 0], pool, bt, lens, out[:, 0], hq, hkv, d, at + R,
                           workspace=workspace(kvhp.q4_decode_workspace_bytes(1, hq, hkv, d, at + R)))
        else:
            kvhp.q4_prefill(q, pool, bt, out, hq, hkv, d, at + R, q_start=pos, seq_lens=lens,
                            workspace=workspace(kvhp.q4_prefill_workspace_bytes(1, R, hq, hkv, d,
                                                                               at + R)))
        outs.append(out)
        qs.append(q)
        at += R
    k, v = (torch.empty((1, hkv, T, d), dtype=torch.float16, device="cuda") for _ in range(2))
    kvhp.q4_gather(pool, bt, torch.tensor([T], dtype=torch.int32, device="cuda"), k, v)
    sync()
    got, q = from_gpu(torch.cat(outs, 1))[0], from_gpu(torch.cat(qs, 1))[0]
    k, v = from_gpu(k)[0].astype(np.float64), from_gpu(v)[0].astype(np.float64)
    G = hq // hkv
    for p in range(T):
        for h in range(hkv):
            hs = slice(h * G, (h + 1) * G)
            o, tol, w, _, _ = attend(q[p, hs], k[h, :p + 1], v[h, :p + 1], np.ones(p + 1, bool))
            # the rows read back were rounded to fp16 once: 2^-11 of each value, and of each
            # product of a score
            size = np.abs(q[p, hs].astype(np.float64)) @ np.abs(k[h, :p + 1]).T / np.sqrt(d)
            tol = tol + (U16 + 2 * U16 * size.max()) * (w @ np.abs(v[h, :p + 1]))
            check(got[p, hs], o, tol, f"position {p} head {h}")
