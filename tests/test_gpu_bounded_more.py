"""Bounded caches past 32-bit offsets, pages that were given away, and calls on
two streams at once, against the definitions in 64 bits."""
import numpy as np
import pytest

import kvhp
from bounded_util import PAGE, Cache, attend, check, decode_ref, plan_ref, workspace
from gpu_util import from_gpu, note, sync, to_gpu
from test_gpu_bounded import (_calls, _check_prefill, _check_sums, _prefill_ref, _prompt_ref,
                              _prompt_weights, _q, _sums, _sums_ref, _weighted, _window_decode,
                              _window_prefill)

pytestmark = pytest.mark.gpu


def _far(c, far_pages):
    """The cache's second half of pages at the end of a pool of far_pages pages per head
    (never written in between); c.near_bt keeps the small pool's ids."""
    import torch
    c.upload()
    n, half = c.pages, c.pages // 2
    pools = []
    for small in (c.pool_k, c.pool_v):
        big = torch.empty((c.hkv, far_pages, PAGE, c.d), dtype=torch.float16, device="cuda")
        big[:, :half].copy_(small[:, :half])
        big[:, far_pages - (n - half):].copy_(small[:, half:])
        pools.append(big)
    c.near_bt = c.bt
    c.bt = np.where(c.bt >= half, c.bt + far_pages - n, c.bt).astype(np.int32)
    c.pages = far_pages
    c.pool_k, c.pool_v = pools
    c.bt_d = to_gpu(c.bt)
    c.kv, c.vv = kvhp.paged_view(pools[0], c.bt_d), kvhp.paged_view(pools[1], c.bt_d)
    return c


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (3, 1, 64)])
def test_pools_past_32_bit_offsets(hq, hkv, d):
    """Pages more than 2^32 bytes behind the start of their head's pool."""
    rng = np.random.default_rng([hq, d])
    c = _far(Cache(rng, [1500, 333], hkv, d), (1 << 32) // (2 * PAGE * d) + 200)
    assert int(c.bt.max()) * PAGE * d * 2 >= 1 << 32
    q = _q(rng, 2, hq, d)
    for window, sinks in [(0, 0), (700, 4), (1100, 20)]:
        note(f"far pages: window_decode window={window}")
        ref, tol, _, _ = decode_ref(q, c, window, sinks)
        check(_window_decode(q, c, window, sinks), ref, tol)
    qp = _q(rng, 2, 20, hq, d)
    start = [1480, 313]
    note("far pages: window_prefill")
    _check_prefill(qp, c, start, 500, 3)
    w, ages = _sums(rng, c)
    note("far pages: weighted_decode")
    out, gw, ga = _weighted(q, c, w, ages, 1, None)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(out, ref, tol)
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 1, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)
    note("far pages: prompt_weights")
    lse, add, rel = _prompt_ref(qp, c, start, 500, 3)
    gw, ga = _prompt_weights(qp, c, lse, w, ages, start, 500, 3, 20)
    rw, tw, ra = _sums_ref(c, w, ages, add, rel, 20, c.lens - 1)
    # keys that no row sees: not touched
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)
    note("far pages: eviction")
    import torch
    budget, moves = 256, torch.zeros(2, hkv, 256, 2, dtype=torch.int32, device="cuda")
    counts = torch.zeros(2, hkv, dtype=torch.int32, device="cuda")
    new = torch.zeros(2, dtype=torch.int32, device="cuda")
    w_d, a_d = to_gpu(gw), to_gpu(ga)
    kvhp.evict_plan(w_d, a_d, c.bt_d, c.lens_d, moves, counts, new, c.cap, budget, 4, 30)
    kvhp.evict_apply(c.pool_k, c.pool_v, w_d, a_d, c.bt_d, moves, counts)
    sync()
    gm, gc = from_gpu(moves), from_gpu(counts)
    crossed = 0
    for b in range(2):
        n = int(c.lens[b])
        pg, sl = c.slots(b)
        ids = torch.from_numpy(pg.astype(np.int64)).cuda()
        ss = torch.from_numpy(sl.astype(np.int64)).cuda()
        for h in range(hkv):
            want = plan_ref(gw[h, pg, sl], ga[h, pg, sl], n, budget, 4, 30, n - 1)
            assert [tuple(x) for x in gm[b, h, :gc[b, h]]] == want
            order = np.arange(n)
            for s, t in want:
                order[t] = s
                crossed += (pg[s] < 1000) != (pg[t] < 1000)
            for pool, host in ((c.pool_k, c.k), (c.pool_v, c.v)):
                # rows gathered page by page: each page is a view with a 64-bit offset
                got = np.stack([from_gpu(pool[h, int(i)])[j] for i, j in zip(pg, sl)])
                assert np.array_equal(got, host[b, h, order])
    assert crossed > 10


def test_prompt_weights_pages_given_away():
    """Entries of pages that no row sees may be -1 or name a page that another sequence took:
    nobody's sums there change but the owner's own."""
    rng = np.random.default_rng(4)
    c = Cache(rng, [640, 700], 2, 64).upload()
    q = _q(rng, 2, 40, 8, 64)
    window, sinks, start = 100, 20, [600, 660]
    w, ages = _sums(rng, c)
    lse, add, rel = _prompt_ref(q, c, start, window, sinks)
    rw, tw, ra = _sums_ref(c, w, ages, add, rel, 40, c.lens - 1)
    bt = c.bt.copy()
    hidden = np.arange(2, (600 - 99) // PAGE)        # behind the sinks, before the window
    bt[0, hidden[::2]] = -1
    bt[0, hidden[1::2]] = bt[1, 40:40 + len(hidden[1::2])].max()   # one of sequence 1's in use
    bt[1, 2] = bt[0, 39]
    c.bt_d.copy_(to_gpu(bt))
    note("prompt_weights over a table with pages given away")
    gw, ga = _prompt_weights(q, c, lse, w, ages, start, window, sinks, 40)
    # the keys of hidden pages: as they were
    for b, pages in ((0, hidden), (1, [2])):
        for i in pages:
            rw[:, c.bt[b, i]], tw[:, c.bt[b, i]] = w[:, c.bt[b, i]], 0
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


def test_two_streams_at_once():
    """Calls that overlap, each with its own workspace and outputs."""
    import torch
    runs = [_calls(np.random.default_rng(s)) for s in (5, 6)]
    wants = []
    note("bounded attention on one stream, then on two at once")
    for go, t, _ in runs:
        go()
        sync()
        wants.append({k: x.clone() for k, x in t.items()})
        for x in t.values():
            x.zero_()
    sync()
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(4):
        for (go, t, _), st in zip(runs, streams):
            with torch.cuda.stream(st):
                t["w"].zero_()
            go(st)
    sync()
    for (_, t, _), want in zip(runs, wants):
        for k, x in t.items():
            assert torch.equal(x, want[k]), k


def test_padded_batches():
    """Rows at negative positions, rows behind the last key, sequences without keys and with
    one, all in one batch: padding keeps what its outputs held."""
    rng = np.random.default_rng(9)
    c = Cache(rng, [0, 1, 16, 90, 300], 2, 128).upload()
    q = _q(rng, 5, 48, 4, 128)
    start = [0, 0, -2 ** 31, 60, 2 ** 31 - 1]
    note("window_prefill over a padded batch")
    _check_prefill(q, c, start, 33, 2)
    w, ages = _sums(rng, c)
    lse, add, rel = _prompt_ref(q, c, start, 33, 2)
    note("prompt_weights over a padded batch")
    gw, ga = _prompt_weights(q, c, lse, w, ages, start, 33, 2, 5)
    rw, tw, ra = _sums_ref(c, w, ages, add, rel, 5, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


@pytest.mark.parametrize("d,visible", [(64, 959), (64, 960), (64, 961), (64, 1029),
                                       (64, 1151), (64, 1152), (64, 1153), (128, 575), (128, 576),
                                       (128, 577), (64, 31), (128, 33)])
@pytest.mark.parametrize("sinks", [0, 1, 17])
def test_window_decode_split_limits(d, visible, sinks):
    """Visible keys on both sides of what one split takes, the window beginning and the first
    tokens ending inside a page; three lengths, one that no gap divides."""
    rng = np.random.default_rng([d, visible, sinks])
    for paged in (True, False):
        c = Cache(rng, [2011, visible, 1300], 2, d, paged=paged).upload()
        q = _q(rng, 3, 14, d)
        note(f"window_decode {visible} visible keys, {sinks} first, d={d} paged={paged}")
        ref, tol, _, _ = decode_ref(q, c, visible - sinks, sinks)
        check(_window_decode(q, c, visible - sinks, sinks), ref, tol)


@pytest.mark.parametrize("n", [5, 127, 128, 129, 160, 447, 448, 449, 703, 704, 705])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (14, 2, 128), (16, 1, 64), (17, 1, 128)])
def test_weighted_decode_split_limits(n, hq, hkv, d):
    """Keys on both sides of what one workgroup a KV head takes, with its sums or without;
    shorter sequences and none beside them."""
    rng = np.random.default_rng([n, hq, d])
    c = Cache(rng, [n, 1, 0, n - 1], hkv, d).upload()
    q = _q(rng, 4, hq, d)
    w, ages = _sums(rng, c)
    note(f"weighted_decode {n} keys, {hq}/{hkv} x {d}")
    out, gw, ga = _weighted(q, c, w, ages, 1, None)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(out, ref, tol)
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 1, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


@pytest.mark.parametrize("hq,hkv", [(71, 1), (33, 1), (12, 4), (2, 2)])
@pytest.mark.parametrize("rows", [1, 3, 17, 33, 63, 64, 65, 130])
def test_prompt_weights_tiles(hq, hkv, rows):
    """Group sizes that no tile of heads divides, rows on both sides of a tile's."""
    rng = np.random.default_rng([hq, rows])
    c = Cache(rng, [rows + 77, max(1, rows - 5)], hkv, 64).upload()
    q = _q(rng, 2, rows, hq, 64)
    start = [77, -3]
    w, ages = _sums(rng, c)
    note(f"prompt_weights {hq}/{hkv}, {rows} rows")
    for window, sinks in [(0, 0), (40, 3)]:
        lse, add, rel = _prompt_ref(q, c, start, window, sinks)
        gw, ga = _prompt_weights(q, c, lse, w, ages, start, window, sinks, rows)
        rw, tw, ra = _sums_ref(c, w, ages, add, rel, rows, c.lens - 1)
        _check_sums(gw, rw, tw)
        assert np.array_equal(ga, ra)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("rows,n,window", [(16, 400, 0), (5, 1500, 0), (16, 4500, 0), (70, 3000, 1200),
                                           (300, 700, 0)])
def test_window_prefill_ranges(hq, hkv, d, rows, n, window):
    """Few rows over many keys: 2 to dozens of ranges, some sequences with fewer than others
    and none, rows enough for either way of joining them."""
    rng = np.random.default_rng([hq, rows, n])
    c = Cache(rng, [n, n // 3, 40], hkv, d).upload()
    q = _q(rng, 3, rows, hq, d)
    note(f"window_prefill {rows} rows over {n} keys, window {window}, {hq}/{hkv} x {d}")
    _check_prefill(q, c, [n - rows, n // 3 - rows, 30], window, 5)


@pytest.mark.parametrize("d", [64, 128])
def test_window_prefill_many_heads_over_ranges(d):
    """More (row, head) pairs than waves run at once, over a few ranges."""
    rng = np.random.default_rng([12, d])
    c = Cache(rng, [900], 16, d).upload()
    q = _q(rng, 1, 260, 32, d)
    note(f"window_prefill 260 rows of 32/16 heads of {d} over 900 keys")
    got, ls = _window_prefill(q, c, [640], 0, 0)
    some = [0, 1, 31, 100, 258, 259]
    ref, tol, lref, ltol = [], [], [], []
    for r in some:
        x = _prefill_ref(q[:, r:r + 1], c, [640 + r], 0, 0)
        for acc, y in zip((ref, tol, lref, ltol), x):
            acc.append(y)
    check(got[:, some], np.concatenate(ref, 1), np.concatenate(tol, 1), "out")
    check(ls[:, :, some], np.concatenate(lref, 2), np.concatenate(ltol, 2), "lse")


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128), (17, 1, 64)])
@pytest.mark.parametrize("n", [30, 639, 641, 959, 961, 1200])
def test_batches_split_limits(n, hq, hkv, d):
    """Batches of 9 ragged sequences on both sides of what one workgroup a KV head takes."""
    rng = np.random.default_rng([n, hq, d])
    c = Cache(rng, [n, 1, 0, n - 1, n // 2, 17, n, n // 3, 64][:9], hkv, d,
              cap=n).upload()
    q = _q(rng, 9, hq, d)
    w, ages = _sums(rng, c)
    note(f"batches: {n} keys, {hq}/{hkv} x {d}")
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(_window_decode(q, c, 0, 0), ref, tol)
    out, gw, ga = _weighted(q, c, w, ages, 1, None)
    check(out, ref, tol)
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 1, np.minimum(c.lens, c.cap) - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


@pytest.mark.parametrize("batch", [7, 15, 16, 17])
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
def test_batches_of_long_sequences(batch, hq, hkv, d):
    """Fixed splits and the batch's own, with sequences of every length beside each other."""
    rng = np.random.default_rng([batch, d])
    lens = rng.integers(0, 2600, batch)
    lens[:3] = [2600, 0, 1]
    c = Cache(rng, lens, hkv, d).upload()
    q = _q(rng, batch, hq, d)
    w, ages = _sums(rng, c)
    note(f"a batch of {batch}, {hq}/{hkv} x {d}")
    ref, tol, _, _ = decode_ref(q, c, 1500, 4)
    check(_window_decode(q, c, 1500, 4), ref, tol)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    out, gw, ga = _weighted(q, c, w, ages, 1, None)
    check(out, ref, tol)
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 1, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


def test_graph_replays_of_short_sequences():
    """One workgroup a KV head with its sums, captured once: each replay adds once more."""
    import torch
    rng = np.random.default_rng(21)
    c = Cache(rng, [300, 17, 0, 101], 2, 64).upload()
    q = to_gpu(_q(rng, 4, 8, 64))
    out = torch.zeros_like(q)
    w = torch.zeros(2, c.pages, PAGE, device="cuda")
    ws = workspace(kvhp.weighted_decode_workspace_bytes(4, 8, 2, 64, 300))

    def go():
        kvhp.weighted_decode(q, c.kv, c.vv, c.lens_d, out, w, 8, 2, 64, 300, new_keys=0,
                             workspace=ws)
    note("weighted_decode of short sequences: eager")
    go()
    sync()
    once, first = w.clone(), out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    w.zero_()
    want = torch.zeros_like(w)
    for i in range(4):
        note(f"replay {i}")
        out.fill_(3)
        sync()
        g.replay()
        sync()
        want += once      # the same fp32 sums in the same order
        assert torch.equal(w, want) and torch.equal(out, first)


@pytest.mark.parametrize("batch,hkv,d,limit", [(3, 2, 64, 832), (3, 8, 64, 896), (6, 8, 64, 1152),
                                               (17, 1, 64, 1152), (2, 2, 128, 544),
                                               (4, 8, 128, 608), (8, 8, 128, 640),
                                               (15, 8, 128, 960), (17, 2, 128, 832),
                                               (16, 8, 128, 960)])
def test_one_split_limits_by_units(batch, hkv, d, limit):
    """Visible keys on both sides of what one split takes, by how many workgroups it makes."""
    rng = np.random.default_rng([batch, hkv, d])
    q = _q(rng, batch, 2 * hkv, d)
    for visible in (limit - 1, limit, limit + 1):
        lens = [visible + 333, visible, 0, visible - 1, visible // 2, 31][:batch]
        lens += list(rng.integers(1, visible + 300, batch - len(lens)))
        for paged in (True, False):
            c = Cache(rng, lens, hkv, d, paged).upload()
            note(f"window_decode: {batch} x {hkv} KV heads of {d}, {visible} visible, paged={paged}")
            ref, tol, _, _ = decode_ref(q, c, visible - 19, 19)
            check(_window_decode(q, c, visible - 19, 19), ref, tol)


@pytest.mark.parametrize("batch,hkv,d,limit", [(3, 2, 64, 768), (3, 8, 64, 896), (6, 8, 64, 960),
                                               (17, 1, 64, 960), (4, 2, 128, 416),
                                               (4, 8, 128, 480), (8, 8, 128, 608),
                                               (17, 2, 128, 832), (16, 8, 128, 960)])
def test_one_split_sums_limits_by_units(batch, hkv, d, limit):
    rng = np.random.default_rng([batch, hkv, d, 1])
    q = _q(rng, batch, 2 * hkv, d)
    for n in (limit - 1, limit, limit + 1):
        lens = [n, n - 1, 0, n // 2, 31, 1][:batch] + list(rng.integers(1, n + 1, max(batch - 6, 0)))
        c = Cache(rng, lens, hkv, d).upload()
        w, ages = _sums(rng, c)
        note(f"weighted_decode: {batch} x {hkv} KV heads of {d}, {n} keys")
        out, gw, ga = _weighted(q, c, w, ages, 2, None)
        ref, tol, sums, rel = decode_ref(q, c, 0, 0)
        check(out, ref, tol)
        rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 2, c.lens - 1)
        _check_sums(gw, rw, tw)
        assert np.array_equal(ga, ra)


def test_steps_over_a_cut_cache_with_rope():
    """Tokens behind an eviction: rotated at their place in the text, appended at their slot,
    attended with what was kept, and cut again."""
    import torch
    rng = np.random.default_rng(31)
    B, hq, hkv, d, n, budget, theta = 3, 8, 2, 64, 150, 96, 10000.0
    c = Cache(rng, [n, n - 30, 40], hkv, d).upload()
    text = c.lens.copy()                       # tokens of the text so far
    pages = c.pages + 6
    pools = [torch.zeros(hkv, pages, PAGE, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    for big, small in zip(pools, (c.pool_k, c.pool_v)):
        big[:, :c.pages] = small
    bt = np.concatenate([c.bt, np.full((B, 1), -1, np.int32)], 1)
    bt[2, 3] = c.pages                         # one more page for the short one
    bt_d = to_gpu(bt)
    kv, vv = kvhp.paged_view(pools[0], bt_d), kvhp.paged_view(pools[1], bt_d)
    w = to_gpu(rng.random((hkv, pages, PAGE)).astype(np.float32))
    ages = torch.zeros(hkv, pages, PAGE, dtype=torch.int32, device="cuda")
    for b in range(B):
        pg, sl = c.slots(b)
        ages[:, to_gpu(pg).long(), to_gpu(sl).long()] = torch.arange(
            int(c.lens[b]), dtype=torch.int32, device="cuda")
    lens, newest = to_gpu(c.lens), to_gpu(text - 1)
    moves = torch.zeros(B, hkv, 96, 2, dtype=torch.int32, device="cuda")
    counts = torch.zeros(B, hkv, dtype=torch.int32, device="cuda")
    new = torch.zeros(B, dtype=torch.int32, device="cuda")
    cap = 10 * PAGE
    ws = workspace(kvhp.weighted_decode_workspace_bytes(B, hq, hkv, d, cap))
    for cut in range(2):
        note(f"cut {cut}: eviction")
        kvhp.evict_plan(w, ages, bt_d, lens, moves, counts, new, cap, budget, 4, 20, newest=newest)
        kvhp.evict_apply(pools[0], pools[1], w, ages, bt_d, moves, counts)
        lens.copy_(new)
        for step in range(5):
            qkv = to_gpu(_q(rng, B, (hq + 2 * hkv) * d))
            q, k, v = (torch.zeros(B, h, d, dtype=torch.float16, device="cuda") for h in (hq, hkv, hkv))
            newest += 1
            text += 1
            note(f"cut {cut}: step {step}")
            kvhp.split_qkv_rope_rows(qkv, B, hq, hkv, d, newest, theta, q, k, v)
            kvhp.paged_append_kv(k, v, pools[0], pools[1], bt_d, lens, B, 1, hkv, d)
            lens += 1
            out = torch.zeros_like(q)
            kvhp.weighted_decode(q, kv, vv, lens, out, w, hq, hkv, d, cap, new_keys=1, ages=ages,
                                 newest=newest, workspace=ws)
            sync()
            slots = from_gpu(lens) - 1
            assert (slots[:2] == budget + step + 0).all() and (from_gpu(newest) == text - 1).all()
            hk, hv, ha = from_gpu(pools[0]), from_gpu(pools[1]), from_gpu(ages)
            for b in range(B):
                # one row at its place in the text, as a prompt's rows are rotated
                one = [torch.zeros(1, h, d, dtype=torch.float16, device="cuda") for h in (hq, hkv, hkv)]
                kvhp.split_qkv_rope(qkv[b:b + 1], 1, hq, hkv, d, int(text[b]) - 1, theta, *one)
                sync()
                m = int(slots[b])
                pg, sl = bt[b, m // PAGE], m % PAGE
                assert torch.equal(one[0][0], q[b])
                assert np.array_equal(hk[:, pg, sl], from_gpu(one[1][0]))
                assert np.array_equal(hv[:, pg, sl], from_gpu(one[2][0]))
                assert (ha[:, pg, sl] == text[b] - 1).all()
                j = np.arange(m + 1)
                hq_ = from_gpu(q[b]).reshape(hkv, -1, d)
                for h in range(hkv):
                    o, tol, _, _, _ = attend(hq_[h], hk[h, bt[b, j // PAGE], j % PAGE],
                                             hv[h, bt[b, j // PAGE], j % PAGE], j >= 0)
                    check(from_gpu(out[b]).reshape(hkv, -1, d)[h], o, tol, f"sequence {b}, head {h}")
                    a = ha[h, bt[b, j // PAGE], j % PAGE]
                    assert len(set(a)) == m + 1 and a.max() == text[b] - 1   # each token once


@pytest.mark.parametrize("d", [64, 128, 96])
def test_prompt_weights_hidden_keys_reach_nothing(d):
    """NaN and infinite K in slots that the window hides from every row, from some, and above
    the diagonal: the sums of keys that the rows see are as without them, and a key's own sum
    is not finite only where a row sees it."""
    rng = np.random.default_rng([d, 77])
    n, rows, window, sinks = 300, 70, 50, 5
    c = Cache(rng, [n, 130], 2, d)
    q = _q(rng, 2, rows, 8, d)
    start = [n - rows, 130 - rows]
    w, ages = _sums(rng, c)
    lse, add, rel = _prompt_ref(q, c, start, window, sinks)
    rw, tw, ra = _sums_ref(c, w, ages, add, rel, 20, c.lens - 1)
    # hidden from every row; seen by the first rows only; by the last only; a first token
    for key in (100, 200, n - 2, 3):
        for bad in (np.nan, np.inf):
            k = c.k.copy()
            c.k[0, :, key] = bad
            c.upload()
            note(f"prompt_weights: K of key {key} is {bad}, d={d}")
            gw, ga = _prompt_weights(q, c, lse, w, ages, start, window, sinks, 20)
            c.k = k
            pg, sl = c.bt[0, key // PAGE], key % PAGE
            hit = gw[:, pg, sl].copy()
            gw[:, pg, sl], want = rw[:, pg, sl], rw.copy()
            _check_sums(gw, want, tw)
            assert np.array_equal(ga, ra)
            if key == 100:
                assert np.array_equal(hit, w[:, pg, sl])      # no row sees it: not touched
            else:
                assert not np.isfinite(hit).any()
