"""The 4-bit cache where its kernels' plans and arithmetic change over: batches of many
sequences, scores that keep growing, pools past 32 bits of bytes, calls on two streams at
once, addresses off 16 bytes (tolerances: bounded_util, q4_util)."""
import numpy as np
import pytest

import kvhp
from bounded_util import PAGE, attend, check, workspace
from gpu_util import from_gpu, note, sync, to_gpu
from q4_util import Q4Cache, quantise, rotated, unpack
from test_gpu_q4 import _check_decode, _check_prefill, _q

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("B,hq,d", [(16, 4, 64), (16, 8, 128), (70, 4, 64), (70, 7, 128), (130, 12, 64),
                                    (64, 16, 128), (33, 3, 64)])
@pytest.mark.parametrize("most", [1, 64, 2500])
def test_decode_of_many_sequences(B, hq, d, most):
    """A few long sequences among short and empty ones; limits on both sides of one split."""
    rng = np.random.default_rng(B + hq + most)
    lens = rng.integers(0, min(most, 150) + 1, B)
    lens[rng.integers(0, B, 2)] = most, 0
    lens[0], lens[-1] = most - most // 7, most
    c = Q4Cache(rng, lens, 1, d).upload()
    q = _q(rng, B, hq, d)
    for cap in (most, 2048, 2049, 9000):
        note(f"q4_decode B={B} {hq}/1 x {d} most={most} cap={cap}")
        c.cap = cap
        _check_decode(q, c, f"cap {cap}")


@pytest.mark.parametrize("n", [768, 769, 1024, 1025, 2048, 2049])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [1, 16])
def test_decode_around_one_split(n, d, B):
    rng = np.random.default_rng(n + d)
    c = Q4Cache(rng, [n] + [5] * (B - 1), 1, d).upload()
    note(f"q4_decode n={n} d={d} B={B}")
    _check_decode(_q(rng, B, 6, d), c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("step", [0.01, 0.2, 3.0, -0.2, -3.0])
def test_scores_that_grow_with_the_key(d, step):
    """Scores that climb (or fall) by `step` a key: a row's largest score moves in every
    tile, by less than fp16's range and by far more."""
    rng = np.random.default_rng(d + int(100 * abs(step)))
    n = 700
    c = Q4Cache(rng, [n], 2, d, slack=0)
    u = rng.choice([-1.0, 1.0], d)
    j = np.zeros((c.pages, PAGE))
    at = np.arange(c.bt.shape[1] * PAGE).reshape(-1, PAGE)
    j[c.bt[0]] = at
    top = 40.0
    # K = u t: q K / sqrt(d) = t with q = u / sqrt(d); past `top`, u's own size grows slowly
    t = np.clip(step * (j - (n if step > 0 else 0)), -top, top)
    kx = (u[None, None, :] * t[..., None] + 0.05 * rng.standard_normal((2, c.pages, PAGE, d))).astype(np.float16)
    kn, kp = quantise(kx)
    c.parts[0], c.parts[1] = kn, np.where(np.isnan(c.parts[1]), c.parts[1], kp)
    c.stand()
    c.upload()
    q = (u / np.sqrt(d) * np.linspace(0.5, 8, 8)[:, None]).astype(np.float16)
    note(f"q4 growing scores step={step} d={d}")
    _check_decode(q[None], c)
    _check_prefill(np.repeat(q[None, None], 300, 1), c, [n - 300], every=23)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("late", [3, 130, 390])
def test_one_key_above_all(d, late):
    """One score far above the others, met first, in the middle and last."""
    rng = np.random.default_rng(d + late)
    c = Q4Cache(rng, [400], 2, d)
    c.parts[1][:, c.bt[0, late // PAGE], late % PAGE, 0] *= np.float16(20)
    c.stand()
    c.upload()
    q = _q(rng, 1, 8, d) * np.float16(3)
    note(f"q4 one key above all at {late}, d={d}")
    _check_decode(q, c)
    _check_prefill(np.repeat(q[:, None], 390, 1), c, [10], every=29)


@pytest.mark.parametrize("B,rows,hq,hkv,d", [(3, 5, 8, 1, 64), (7, 40, 8, 2, 128), (64, 3, 4, 1, 64),
                                             (65, 3, 4, 1, 64), (5, 130, 7, 1, 128), (16, 9, 20, 1, 64)])
def test_chunks_of_many_sequences(B, rows, hq, hkv, d):
    """Ranges of keys shared out by ragged lengths: long sequences among short ones and
    empty ones, one long one alone, all as long as can be."""
    rng = np.random.default_rng(B + rows)
    most = 2600
    for kind in ("ragged", "one", "all"):
        lens = rng.integers(0, 150, B)
        lens[rng.integers(0, B, 2)] = most, 0
        if kind == "one":
            lens[:] = rows
            lens[B // 2] = most
        elif kind == "all":
            lens[:] = most if B < 16 else 1300
        c = Q4Cache(rng, lens, hkv, d).upload()
        note(f"q4_prefill B={B} rows={rows} {hq}/{hkv} x {d} {kind}")
        q = _q(rng, B, rows, hq, d)
        _check_prefill(q, c, np.asarray(lens) - rows, kind, every=17)
        c.cap = 9000 if kind == "one" else 1000   # a limit above and below the lengths
        _check_prefill(q, c, np.asarray(lens) - rows, f"{kind} cap", every=17)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 8), (6, 2, 24), (8, 1, 56), (32, 2, 72), (6, 6, 80), (14, 2, 96),
                                      (8, 2, 112), (20, 1, 136), (4, 1, 160), (3, 1, 192), (34, 2, 200),
                                      (8, 2, 248), (4, 2, 256)])
def test_any_head_dim(hq, hkv, d):
    """Tokens, chunks and prompts over ragged lengths, with ranges of keys and without."""
    rng = np.random.default_rng(hq + d)
    c = Q4Cache(rng, [1500, 0, 77, 64, 1], hkv, d).upload()
    note(f"q4_decode {hq}/{hkv} x {d}")
    _check_decode(_q(rng, 5, hq, d), c)
    note("chunks")
    _check_prefill(_q(rng, 5, 11, hq, d), c, [1489, 0, 66, 60, -3], every=3)
    note("a prompt")
    c = Q4Cache(rng, [150, 131], hkv, d).upload()
    _check_prefill(_q(rng, 2, 150, hq, d), c, None, every=31)
    note("steep scores and rows of many sizes")
    c = Q4Cache(rng, [300], hkv, d, scale=3.0, offset=20.0)
    c.parts[3][:, ::2, ::3, 0] *= np.float16(50)
    c.parts[3][:, 1::2, ::2, 0] *= np.float16(1e-4)
    c.parts[3][:, :, 5, 0] *= np.float16(-1)
    c.stand()
    c.upload()
    _check_decode(_q(rng, 1, hq, d), c)
    _check_prefill(_q(rng, 1, 40, hq, d), c, [260], every=7)


@pytest.mark.parametrize("d", [64, 96, 128])
def test_chunks_off_16_bytes(d):
    """More rows than one wave takes, q and out off their alignment, over ranges of keys."""
    rng = np.random.default_rng(d)
    c = Q4Cache(rng, [1900, 60], 2, d).upload()
    x = _q(rng, 2, 30, 8, d)
    q = torch.empty(x.size + 1, dtype=torch.float16, device="cuda")[1:].view(x.shape)
    q.copy_(to_gpu(x))
    out = torch.full((x.size + 1,), 7.0, dtype=torch.float16, device="cuda")[1:].view(x.shape)
    note(f"q4_prefill off 16 bytes d={d}")
    kvhp.q4_prefill(q, c.pool, c.bt_d, out, 8, 2, d, c.cap, q_start=to_gpu(np.array([1870, 40], np.int32)),
                    seq_lens=c.lens_d,
                    workspace=workspace(kvhp.q4_prefill_workspace_bytes(2, 30, 8, 2, d, c.cap)))
    sync()
    got = from_gpu(out)
    assert (got[1, 20:] == 7).all()
    for b, first, rows in ((0, 1870, 30), (1, 40, 20)):
        for r in range(0, rows, 6):
            for h in range(2):
                n, hs = first + r + 1, slice(4 * h, 4 * h + 4)
                o, tol, _, _, _ = attend(x[b, r, hs], c.k[b, h, :n], c.v[b, h, :n], np.ones(n, bool))
                check(got[b, r, hs], o, tol, f"sequence {b} row {r} head {h}")


@pytest.mark.parametrize("d", [96, 128])
def test_pools_past_32_bits(d):
    """Pages of more than 4 GiB per head: the bits of the same rows in a small pool."""
    rng = np.random.default_rng(9)
    hq, hkv, n = 8, 2, 400
    pages = (n + PAGE - 1) // PAGE
    rows = to_gpu(_q(rng, 1, n, hq + 2 * hkv, d))
    parts = [rows[:, :, :hq], rows[:, :, hq:hq + hkv], rows[:, :, hq + hkv:]]
    lens = to_gpu(np.array([n], np.int32))
    got = []
    for many in (pages, (1 << 32) // kvhp.q4_page_bytes(d) + 5000):
        ids = np.arange(many - pages, many)[::-1].astype(np.int32)
        bt = to_gpu(ids[None].copy())
        pool = torch.empty((hkv, many, kvhp.q4_page_bytes(d)), dtype=torch.uint8, device="cuda")
        q = torch.empty((1, n, hq, d), dtype=torch.float16, device="cuda")
        note(f"q4 pool of {many} pages: append")
        kvhp.q4_rope_append(*parts, None, q, pool, bt, hq, hkv, d, 10000.0)
        back = [torch.empty((1, hkv, n, d), dtype=torch.float16, device="cuda") for _ in range(2)]
        note("gather")
        kvhp.q4_gather(pool, bt, lens, *back)
        out = torch.empty_like(q)
        note("prefill")
        kvhp.q4_prefill(q, pool, bt, out, hq, hkv, d, n,
                        workspace=workspace(kvhp.q4_prefill_workspace_bytes(1, n, hq, hkv, d, n)))
        few = torch.empty((1, 5, hq, d), dtype=torch.float16, device="cuda")
        note("prefill of few rows")
        kvhp.q4_prefill(q[:, -5:].contiguous(), pool, bt, few, hq, hkv, d, n, q_start=lens - 5,
                        workspace=workspace(kvhp.q4_prefill_workspace_bytes(1, 5, hq, hkv, d, n)))
        one = torch.empty((1, hq, d), dtype=torch.float16, device="cuda")
        note("decode")
        kvhp.q4_decode(q[:, -1].contiguous(), pool, bt, lens, one, hq, hkv, d, n,
                       workspace=workspace(kvhp.q4_decode_workspace_bytes(1, hq, hkv, d, n)))
        sync()
        got.append([t.clone() for t in (q, *back, out, few, one)])
        del pool
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.isfinite(got[0][3]).all()


def test_fp16_pools_past_32_bits():
    rng = np.random.default_rng(10)
    hkv, d, n = 2, 128, 40
    many = (1 << 32) // (PAGE * d * 2) + 100
    rows = to_gpu(_q(rng, 1, n, 2 * hkv, d))
    pk, pv = (torch.empty((hkv, many, PAGE, d), dtype=torch.float16, device="cuda") for _ in range(2))
    ids = np.array([[many - 1, 7, many - 3]], np.int32)
    note("rope_append past 4 GiB")
    kvhp.rope_append(None, rows[:, :, :hkv], rows[:, :, hkv:], None, None, pk, pv, to_gpu(ids), hkv, hkv, d, 0.0)
    sync()
    for pool, x in ((pk, rows[0, :, :hkv]), (pv, rows[0, :, hkv:])):
        got = torch.cat([pool[:, int(i)] for i in ids[0]], 1)[:, :n]
        assert torch.equal(got, x.transpose(0, 1))


def test_two_streams_at_once():
    """Calls that overlap, each with its own workspace, output and pool."""
    rng = np.random.default_rng(13)
    sets = []
    for i, lens in enumerate(([4000, 3000], [3500, 10])):
        c = Q4Cache(rng, lens, 2, 128).upload()
        q = to_gpu(_q(rng, 2, 40, 8, 128))
        start = to_gpu(np.maximum(np.asarray(lens, np.int32) - 40, 0))
        ws = [workspace(kvhp.q4_decode_workspace_bytes(2, 8, 2, 128, c.cap)),
              workspace(kvhp.q4_prefill_workspace_bytes(2, 40, 8, 2, 128, c.cap))]
        sets.append((c, q, start, ws, torch.cuda.Stream()))

    def run(c, q, start, ws, out, one):
        kvhp.q4_prefill(q, c.pool, c.bt_d, out, 8, 2, 128, c.cap, q_start=start, seq_lens=c.lens_d,
                        workspace=ws[1])
        kvhp.q4_decode(out[:, 0].contiguous(), c.pool, c.bt_d, c.lens_d, one, 8, 2, 128, c.cap,
                       workspace=ws[0])

    def outs():
        return (torch.zeros((2, 40, 8, 128), dtype=torch.float16, device="cuda"),
                torch.zeros((2, 8, 128), dtype=torch.float16, device="cuda"))

    note("q4 streams: one after the other")
    want = []
    for c, q, start, ws, _ in sets:
        o = outs()
        run(c, q, start, ws, *o)
        sync()
        want.append(o)
    got = [[outs() for _ in range(6)] for _ in sets]
    sync()
    note("q4 streams: overlapping")
    for i in range(6):
        for (c, q, start, ws, side), o in zip(sets, got):
            with torch.cuda.stream(side):
                run(c, q, start, ws, *o[i])
    sync()
    for w, g in zip(want, got):
        for o in g:
            assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


@pytest.mark.parametrize("d", [64, 128])
def test_addresses_off_16_bytes(d):
    """Queries and outputs that begin at an odd element."""
    rng = np.random.default_rng(d)
    c = Q4Cache(rng, [150, 0, 33], 2, d).upload()
    x = _q(rng, 3, 8, d)
    q = torch.empty(x.size + 1, dtype=torch.float16, device="cuda")[1:].view(x.shape)
    q.copy_(to_gpu(x))
    out = torch.full((x.size + 2,), 7.0, dtype=torch.float16, device="cuda")
    note(f"q4 off 16 bytes d={d}")
    kvhp.q4_decode(q, c.pool, c.bt_d, c.lens_d, out[1:-1].view(x.shape), 8, 2, d, c.cap,
                   workspace=workspace(kvhp.q4_decode_workspace_bytes(3, 8, 2, d, c.cap)))
    sync()

    def holds(got, what):
        assert got[0] == 7 and got[-1] == 7
        got = got[1:-1].reshape(x.shape)
        for b in (0, 2):
            for h in range(2):
                n, hs = int(c.lens[b]), slice(4 * h, 4 * h + 4)
                o, tol, _, _, _ = attend(x[b, hs], c.k[b, h, :n], c.v[b, h, :n], np.ones(n, bool))
                check(got[b, hs], o, tol, f"{what} {b} {h}")
        return got[1]

    assert (holds(from_gpu(out), "decode") == 0).all()
    out.fill_(7)
    kvhp.q4_prefill(q[:, None], c.pool, c.bt_d, out[1:-1].view((3, 1, 8, d)), 8, 2, d, c.cap,
                    q_start=to_gpu(np.array([149, 0, 32], np.int32)), seq_lens=c.lens_d,
                    workspace=workspace(kvhp.q4_prefill_workspace_bytes(3, 1, 8, 2, d, c.cap)))
    sync()
    assert (holds(from_gpu(out), "prefill") == 7).all()


def test_more_sequences_than_a_grid_axis_of_splits():
    """5000 sequences that might have 16384 keys each."""
    rng = np.random.default_rng(50)
    B, d = 5000, 64
    c = Q4Cache(rng, rng.integers(0, 40, B), 1, d, cap=16384).upload()
    note(f"q4_decode B={B}")
    _check_decode(_q(rng, B, 2, d), c)


@pytest.mark.parametrize("d", [40, 64, 128])
def test_positions_before_the_text(d):
    """Negative positions rotate the other way, if their slots are not."""
    rng = np.random.default_rng(d)
    hq, hkv, R = 4, 2, 9
    x = _q(rng, 2, R, hq + 2 * hkv, d)
    t = to_gpu(x)
    pos, slots = np.array([-5, -(1 << 31)], np.int32), np.array([0, 3], np.int32)
    pk, pv = (torch.zeros((hkv, 2, PAGE, d), dtype=torch.float16, device="cuda") for _ in range(2))
    q = torch.zeros((2, R, hq, d), dtype=torch.float16, device="cuda")
    note(f"rope_append at negative positions d={d}")
    kvhp.rope_append(t[:, :, :hq], t[:, :, hq:hq + hkv], t[:, :, hq + hkv:], to_gpu(pos), q, pk, pv,
                     to_gpu(np.array([[0], [1]], np.int32)), hq, hkv, d, 10000.0, slots=to_gpu(slots))
    sync()
    at = (pos[:, None].astype(np.int64) + np.arange(R))[..., None]
    want, e = rotated(x[:, :, :hq], at, 10000.0)
    assert (np.abs(from_gpu(q) - want) <= np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + e * 1.01).all()
    want, e = rotated(x[:, :, hq:hq + hkv], at, 10000.0)
    got = from_gpu(pk)
    for b in range(2):
        g = got[:, b, slots[b]:slots[b] + R].transpose(1, 0, 2)
        assert (np.abs(g - want[b]) <= np.abs(want[b]) * 2.0 ** -11 + 2.0 ** -25 + e[b] * 1.01).all()
        assert np.array_equal(from_gpu(pv)[:, b, slots[b]:slots[b] + R].transpose(1, 0, 2), x[b, :, hq + hkv:])


@pytest.mark.parametrize("hq,hkv", [(16380, 2), (16381, 2), (4, 9000)])
def test_append_of_many_heads(hq, hkv):
    """Both sides of the most heads a workgroup's rows are counted for."""
    rng = np.random.default_rng(hq)
    d, R = 64, 3
    x = _q(rng, 1, R, hq + 2 * hkv, d)
    t = to_gpu(x)
    pool = torch.zeros((hkv, 1, kvhp.q4_page_bytes(d)), dtype=torch.uint8, device="cuda")
    q = torch.zeros((1, R, hq, d), dtype=torch.float16, device="cuda")
    bt = to_gpu(np.zeros((1, 1), np.int32))
    note(f"q4_rope_append {hq}/{hkv} heads")
    kvhp.q4_rope_append(t[:, :, :hq], t[:, :, hq:hq + hkv], t[:, :, hq + hkv:], None, q, pool, bt,
                        hq, hkv, d, 10000.0)
    sync()
    want, e = rotated(x[:, :, :hq], np.arange(R)[None, :, None], 10000.0)
    assert (np.abs(from_gpu(q) - want) <= np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + e * 1.01).all()
    _, _, vn, vp = unpack(from_gpu(pool), d)
    n, p = quantise(x[0, :, hq + hkv:].transpose(1, 0, 2))
    assert np.array_equal(vn[:, 0, :R], n) and np.array_equal(vp[:, 0, :R], p)


@pytest.mark.parametrize("d", [64, 96, 128])
def test_replays_follow_the_lengths(d):
    """Lengths and starts are read where the kernels run: a captured step and a captured chunk
    over lengths that change between replays, against eager calls, bit for bit."""
    rng = np.random.default_rng(d)
    B, rows, hq, hkv = 18, 40, 8, 2
    most = 2600
    c = Q4Cache(rng, [most] * B, hkv, d).upload()
    q, x = to_gpu(_q(rng, B, hq, d)), to_gpu(_q(rng, 4, rows, hq, d))
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    start = torch.zeros(4, dtype=torch.int32, device="cuda")
    bt4 = c.bt_d[:4].contiguous()

    def buffers():
        return (torch.zeros_like(q), torch.zeros_like(x), torch.zeros((4, hq, rows), device="cuda"),
                workspace(kvhp.q4_decode_workspace_bytes(B, hq, hkv, d, most)),
                workspace(kvhp.q4_prefill_workspace_bytes(4, rows, hq, hkv, d, most)))

    def run(one, out, lse, dws, pws):
        kvhp.q4_decode(q, c.pool, c.bt_d, lens, one, hq, hkv, d, most, workspace=dws)
        kvhp.q4_prefill(x, c.pool, bt4, out, hq, hkv, d, most, q_start=start, seq_lens=lens[:4], lse=lse,
                        workspace=pws)

    got = buffers()
    graph = torch.cuda.CUDAGraph()
    note(f"q4 capture d={d}")
    with torch.cuda.graph(graph):
        run(*got)
    for i, new in enumerate(([most] * B, [40] * B, list(rng.integers(0, most + 1, B)), [most] + [0] * (B - 1))):
        note(f"q4 replay {i} d={d}")
        lens.copy_(to_gpu(np.asarray(new, np.int32)))
        start.copy_(lens[:4] - rows)
        for t in got[:3]:
            t.fill_(3)
        graph.replay()
        sync()
        want = buffers()
        for t in want[:3]:
            t.fill_(3)
        run(*want)
        sync()
        assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
        assert torch.isfinite(got[0]).all() and (i > 0 or not (got[1] == 3).all())
