"""Attention over a bounded cache and the sums of attention weight, against
their definitions in 64 bits (tolerances: bounded_util)."""
import math

import numpy as np
import pytest

import kvhp
from bounded_util import (PAGE, U16, U32, Cache, attend, check, decode_ref, visible, workspace)
from gpu_util import from_gpu, note, sync, to_gpu

pytestmark = pytest.mark.gpu


def _q(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


def _window_decode(q, c, window, sinks, max_len=None, stream=None, out=None):
    import torch
    B, hq, d = q.shape
    max_len = c.cap if max_len is None else max_len
    ws = workspace(kvhp.window_decode_workspace_bytes(B, hq, c.hkv, d, max_len, window, sinks))
    q_d = to_gpu(q)
    if out is None:
        out = torch.full(q.shape, math.nan, dtype=torch.float16, device="cuda")
    kvhp.window_decode(q_d, c.kv, c.vv, c.lens_d, out, hq, c.hkv, d, max_len, window, sinks,
                       workspace=ws, stream=stream)
    sync()
    return from_gpu(out)


HEADS = [(32, 8, 128), (8, 2, 64), (14, 2, 64), (4, 4, 128), (16, 1, 64), (6, 2, 128),
         (20, 1, 64), (24, 1, 128), (6, 3, 80), (2, 1, 256), (3, 1, 33)]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_window_decode_heads(hq, hkv, d, paged):
    rng = np.random.default_rng([hq, hkv, d])
    c = Cache(rng, [300, 1, 0, 77, 130], hkv, d, paged).upload()
    q = _q(rng, 5, hq, d)
    for window, sinks in [(50, 4), (0, 0), (128, 37)]:
        note(f"window_decode {hq}/{hkv} x {d} paged={paged} window={window} sinks={sinks}")
        ref, tol, _, _ = decode_ref(q, c, window, sinks)
        check(_window_decode(q, c, window, sinks), ref, tol, f"window={window}")


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 16), (15, 3), (16, 16), (17, 15),
                                          (31, 33), (64, 0), (100, 500), (1000, 7), (0, 9)])
def test_window_decode_edges(window, sinks, paged):
    """Every length around a page and a step, windows and sinks that meet, cross and overlap."""
    rng = np.random.default_rng([window, sinks])
    lens = [1, 2, 3, 15, 16, 17, 18, 31, 32, 33, 47, 48, 49, 63, 64, 65, 66, 95, 97, 128, 129, 200,
            513, 0]
    c = Cache(rng, lens, 2, 64, paged).upload()
    q = _q(rng, len(lens), 8, 64)
    note(f"window_decode edges window={window} sinks={sinks} paged={paged}")
    ref, tol, _, _ = decode_ref(q, c, window, sinks)
    check(_window_decode(q, c, window, sinks), ref, tol)


@pytest.mark.parametrize("batch,ctx,window,sinks", [(1, 5000, 2048, 4), (1, 9001, 0, 0),
                                                    (9, 3000, 1500, 20), (33, 700, 333, 5),
                                                    (2, 20000, 12345, 100)])
def test_window_decode_long(batch, ctx, window, sinks):
    """Contexts that split into many parts, whose join carries the maximum and the sum."""
    rng = np.random.default_rng([batch, ctx])
    lens = rng.integers(1, ctx + 1, batch)
    lens[-1] = ctx
    c = Cache(rng, lens, 2, 128, scale=1.5).upload()
    q = _q(rng, batch, 8, 128, scale=1.5)
    note(f"window_decode long {batch} x {ctx} window={window} sinks={sinks}")
    ref, tol, _, _ = decode_ref(q, c, window, sinks)
    check(_window_decode(q, c, window, sinks), ref, tol)


@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("paged", [True, False])
def test_window_decode_hidden_slots_reach_nothing(d, paged):
    """NaN and infinite rows in hidden slots, in pages that visible keys share too, and
    table entries of hidden pages that name no page or another sequence's."""
    rng = np.random.default_rng(d)
    lens, window, sinks = [400, 150, 52, 16], 45, 5
    c = Cache(rng, lens, 2, d, paged)
    q = _q(rng, 4, 8, d)
    ref, tol, _, _ = decode_ref(q, c, window, sinks)
    for b, n in enumerate(lens):
        hidden = ~visible(n - 1, n, window, sinks)
        bad = np.array([np.nan, np.inf, -np.inf], np.float16)[np.arange(hidden.sum()) % 3]
        c.k[b][:, np.flatnonzero(hidden)] = bad[None, :, None]
        c.v[b][:, np.flatnonzero(hidden)] = bad[None, :, None]
    if paged:
        c.upload()   # pages uploaded, then their entries lost
        see = visible(399, 400, window, sinks)
        for i in range(400 // PAGE):
            if not see[PAGE * i:PAGE * (i + 1)].any():
                c.bt[0, i] = -1 if i % 2 else 10 ** 6
        c.bt_d.copy_(to_gpu(c.bt))
    else:
        c.upload()
    note(f"window_decode hidden d={d} paged={paged}")
    check(_window_decode(q, c, window, sinks), ref, tol)


def test_window_decode_strides_and_capacity():
    """Rows 8 elements apart from packed, views that start inside an allocation, unaligned
    tensors, and lengths above max_seq_len."""
    import torch
    rng = np.random.default_rng(3)
    lens, hkv, d, window, sinks = np.array([200, 90], np.int32), 2, 64, 70, 6
    q = _q(rng, 2, 8, d)
    for pad, shift in [(8, 0), (8, 8), (3, 1), (0, 4)]:
        note(f"window_decode strides pad={pad} shift={shift}")
        c = Cache(rng, lens, hkv, d, False).upload()
        T, pitch = 200, d + pad
        held = []
        for name in ("k", "v"):
            flat = torch.full((shift + 2 * hkv * T * pitch,), math.nan, dtype=torch.float16,
                              device="cuda")
            x = flat[shift:].view(2, hkv, T, pitch)
            x[..., :d] = to_gpu(getattr(c, name))
            held.append(x)
        c.kv, c.vv = (kvhp.strided_view(x, hkv * T * pitch, T * pitch, pitch) for x in held)
        ref, tol, _, _ = decode_ref(q, c, window, sinks)
        check(_window_decode(q, c, window, sinks), ref, tol)
    c = Cache(rng, lens, hkv, d).upload()
    c.cap = 120
    note("window_decode lengths above max_seq_len")
    ref, tol, _, _ = decode_ref(q, c, window, sinks)
    check(_window_decode(q, c, window, sinks), ref, tol)


# ------------------------------------------------------------ prompt rows --
def _prefill_ref(q, c, start, window, sinks):
    B, R, hq, d = q.shape
    G = hq // c.hkv
    out, tol = np.full(q.shape, 7.0), np.zeros(q.shape)
    lse, ltol = np.full((B, hq, R), 7.0), np.zeros((B, hq, R))
    for b in range(B):
        n = min(int(c.lens[b]), c.cap)
        for r in range(R):
            p = int(start[b]) + r
            if p < 0 or p >= n:
                continue
            see = visible(p, n, window, sinks)
            for h in range(c.hkv):
                hs = slice(h * G, (h + 1) * G)
                with np.errstate(invalid="ignore"):
                    out[b, r, hs], tol[b, r, hs], _, lse[b, hs, r], ds = attend(
                        q[b, r, hs], c.k[b, h, :n], c.v[b, h, :n], see)
                ltol[b, hs, r] = ds + (see.sum() + 8) * U32 + 4 * U32 * abs(lse[b, hs, r])
    return out, tol, lse, ltol


def _window_prefill(q, c, start, window, sinks, lse=True, stream=None):
    import torch
    B, R, hq, d = q.shape
    ws = workspace(kvhp.window_prefill_workspace_bytes(B, R, hq, c.hkv, d, c.cap, window, sinks))
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    ls = torch.full((B, hq, R), 7.0, device="cuda") if lse else None
    kvhp.window_prefill(to_gpu(q), c.kv, c.vv, out, hq, c.hkv, d, c.cap, window, sinks,
                        q_start=None if start is None else to_gpu(np.asarray(start, np.int32)),
                        seq_lens=c.lens_d, lse=ls, workspace=ws, stream=stream)
    sync()
    return from_gpu(out), None if ls is None else from_gpu(ls)


def _check_prefill(q, c, start, window, sinks):
    got, ls = _window_prefill(q, c, start, window, sinks)
    ref, tol, lref, ltol = _prefill_ref(q, c, [0] * len(q) if start is None else start, window,
                                        sinks)
    check(got, ref, tol, "out")
    check(ls, lref, ltol, "lse")


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_window_prefill_heads(hq, hkv, d, paged):
    rng = np.random.default_rng([hq, hkv, d, 1])
    R = 90
    c = Cache(rng, [90, 41, 0], hkv, d, paged).upload()
    q = _q(rng, 3, R, hq, d)
    for window, sinks in [(20, 3), (0, 0)]:
        note(f"window_prefill {hq}/{hkv} x {d} paged={paged} window={window} sinks={sinks}")
        _check_prefill(q, c, None, window, sinks)


@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 64, 65, 127, 200])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (64, 64), (65, 63), (100, 300), (0, 2)])
def test_window_prefill_chunks(rows, window, sinks):
    """Chunks behind cached keys, at the end and inside a sequence, and some of whose rows lie
    before the first key or behind the last."""
    rng = np.random.default_rng([rows, window, sinks])
    lens = [400, rows, max(1, rows - 3), 290]
    c = Cache(rng, lens, 2, 64).upload()
    q = _q(rng, 4, rows, 8, 64)
    note(f"window_prefill chunk rows={rows} window={window} sinks={sinks}")
    _check_prefill(q, c, [400 - rows, 0, -3, 290 - rows // 2 - 1], window, sinks)


@pytest.mark.parametrize("S,window,sinks,heads", [(600, 130, 5, (8, 2, 128)),
                                                  (515, 0, 0, (14, 2, 64)),
                                                  (1030, 700, 20, (8, 2, 64))])
def test_window_prefill_prompts(S, window, sinks, heads):
    hq, hkv, d = heads
    rng = np.random.default_rng(S)
    c = Cache(rng, [S, S - 77], hkv, d, False, scale=1.5).upload()
    q = _q(rng, 2, S, hq, d, scale=1.5)
    note(f"window_prefill prompt S={S} window={window} sinks={sinks} heads={heads}")
    _check_prefill(q, c, None, window, sinks)


def test_window_prefill_few_rows_long_cache():
    """A few rows over a long cache, whose keys are read in parts."""
    rng = np.random.default_rng(11)
    c = Cache(rng, [5000, 3111], 2, 128).upload()
    q = _q(rng, 2, 9, 8, 128)
    for window, sinks in [(0, 0), (2500, 30)]:
        note(f"window_prefill 9 rows behind 5000 keys, window={window}")
        _check_prefill(q, c, [4991, 3102], window, sinks)


@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("paged", [True, False])
def test_window_prefill_hidden_values_reach_nothing(d, paged):
    """A key's infinite or NaN V (and K) reaches the rows that see it and no other: above the
    diagonal, behind the window, and between the sinks and the window."""
    rng = np.random.default_rng([d, 5])
    S, window, sinks = 200, 40, 6
    c = Cache(rng, [S], 2, d, paged)
    q = _q(rng, 1, S, 8, d)
    ref, tol, lref, ltol = _prefill_ref(q, c, [0], window, sinks)
    for key, bad in [(70, np.nan), (133, np.inf), (50, -np.inf), (5, np.nan)]:
        v, k = c.v.copy(), c.k.copy()
        c.v[:, :, key] = bad
        c.upload()
        note(f"window_prefill hidden V d={d} paged={paged} key={key}")
        got, ls = _window_prefill(q, c, None, window, sinks)
        sees = np.array([visible(p, S, window, sinks)[key] for p in range(S)])
        check(got[:, ~sees], ref[:, ~sees], tol[:, ~sees], f"V of key {key}")
        check(ls, lref, ltol, "lse")
        hit = got[:, sees]
        assert np.isnan(hit).all() if np.isnan(bad) else (hit == bad).all()
        c.v = v
        c.k[:, :, key] = np.nan
        c.upload()
        got, ls = _window_prefill(q, c, None, window, sinks)
        check(got[:, ~sees], ref[:, ~sees], tol[:, ~sees], f"K of key {key}")
        check(ls[:, :, ~sees], lref[:, :, ~sees], ltol[:, :, ~sees], "lse")
        assert np.isnan(got[:, sees]).all()
        c.k = k


def test_window_prefill_equals_decode_and_lse_is_optional():
    rng = np.random.default_rng(21)
    c = Cache(rng, [333], 2, 64).upload()
    q = _q(rng, 1, 1, 8, 64)
    note("window_prefill one row against window_decode")
    a, _ = _window_prefill(q, c, [332], 100, 4)
    b, ls = _window_prefill(q, c, [332], 100, 4, lse=False)
    assert ls is None and np.array_equal(a, b)
    ref, tol, _, _ = decode_ref(q[:, 0], c, 100, 4)
    check(a[:, 0], ref, tol)


def test_window_prefill_only_needed_pages():
    """Table entries of pages that no row of the chunk sees are not read."""
    rng = np.random.default_rng(22)
    window, sinks, R, n = 50, 3, 40, 500
    c = Cache(rng, [n], 2, 64)
    q = _q(rng, 1, R, 8, 64)
    ref, tol, lref, ltol = _prefill_ref(q, c, [n - R], window, sinks)
    see = np.any([visible(p, n, window, sinks) for p in range(n - R, n)], axis=0)
    c.k[:, :, ~see], c.v[:, :, ~see] = np.nan, np.inf
    c.upload()
    for i in range(n // PAGE):
        if not see[PAGE * i:PAGE * (i + 1)].any():
            c.bt[0, i] = -1 if i % 2 else 10 ** 6
    c.bt_d.copy_(to_gpu(c.bt))
    note("window_prefill with lost pages")
    got, ls = _window_prefill(q, c, [n - R], window, sinks)
    check(got, ref, tol)
    check(ls, lref, ltol)


# ------------------------------------------------------------------- sums --
def _sums(rng, c):
    w = rng.random((c.hkv, c.pages, PAGE)).astype(np.float32)
    w[rng.random(w.shape) < 0.05] = np.nan          # stale slots
    for b in range(len(c.lens)):
        pg, sl = c.slots(b)
        w[:, pg, sl] = rng.random((c.hkv, len(pg)))
    return w, rng.integers(0, 1000, w.shape).astype(np.int32)


def _sums_ref(c, w, ages, add, rel, new_keys, newest):
    """Expected sums, their tolerance and ages after adding add[b, h] [n]."""
    ref, tol, age = w.astype(np.float64), np.zeros(w.shape), ages.copy()
    for b in range(len(c.lens)):
        n = min(int(c.lens[b]), c.cap)
        pg, sl = (x[:n] for x in c.slots(b))
        f = max(0, n - new_keys)
        for h in range(c.hkv):
            if (b, h) not in add:
                continue
            x = add[b, h]
            t = rel[b, h] * x + 2.0 ** -120
            ref[h, pg[:f], sl[:f]] += x[:f]
            ref[h, pg[f:], sl[f:]] = x[f:]
            tol[h, pg, sl] = t + U32 * np.abs(ref[h, pg, sl])
            age[h, pg[f:], sl[f:]] = newest[b] - (n - 1 - np.arange(f, n))
    return ref, tol, age


def _check_sums(got, ref, tol):
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    live = ~np.isnan(ref)
    check(got[live], ref[live], tol[live], "weights")


def _weighted(q, c, w, ages, new_keys, newest, stream=None):
    import torch
    B, hq, d = q.shape
    ws = workspace(kvhp.weighted_decode_workspace_bytes(B, hq, c.hkv, d, c.cap))
    out = torch.full(q.shape, math.nan, dtype=torch.float16, device="cuda")
    w_d, a_d = to_gpu(w), None if ages is None else to_gpu(ages)
    kvhp.weighted_decode(to_gpu(q), c.kv, c.vv, c.lens_d, out, w_d, hq, c.hkv, d, c.cap,
                         new_keys=new_keys, ages=a_d,
                         newest=None if newest is None else to_gpu(np.asarray(newest, np.int32)),
                         workspace=ws, stream=stream)
    sync()
    return from_gpu(out), from_gpu(w_d), None if a_d is None else from_gpu(a_d)


@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_weighted_decode_heads(hq, hkv, d):
    rng = np.random.default_rng([hq, hkv, d, 2])
    c = Cache(rng, [300, 1, 0, 77, 130], hkv, d).upload()
    q = _q(rng, 5, hq, d)
    w, ages = _sums(rng, c)
    newest = c.lens + 100
    note(f"weighted_decode {hq}/{hkv} x {d}")
    out, gw, ga = _weighted(q, c, w, ages, 1, newest)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(out, ref, tol, "out")
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, 1, newest)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


@pytest.mark.parametrize("batch,ctx", [(1, 64), (1, 65), (1, 3000), (3, 9000), (8, 1000),
                                       (40, 600), (9, 5000)])
@pytest.mark.parametrize("new_keys", [0, 1, 17, 10 ** 9])
def test_weighted_decode_lengths(batch, ctx, new_keys):
    rng = np.random.default_rng([batch, ctx])
    lens = rng.integers(1, ctx + 1, batch)
    lens[0] = ctx
    c = Cache(rng, lens, 2, 64).upload()
    q = _q(rng, batch, 8, 64)
    w, ages = _sums(rng, c)
    note(f"weighted_decode {batch} x {ctx} new_keys={new_keys}")
    out, gw, ga = _weighted(q, c, w, ages, new_keys, None)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(out, ref, tol, "out")
    rw, tw, ra = _sums_ref(c, w, ages, sums, rel, new_keys, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)
    _, gw2, _ = _weighted(q, c, w, None, new_keys, None)   # without ages: the same sums
    assert np.array_equal(gw, gw2, equal_nan=True)


def test_weighted_decode_bad_pages():
    """Ids outside the pool: read as the pool's nearest page, their sums dropped."""
    rng = np.random.default_rng(8)
    c = Cache(rng, [100], 2, 64)
    last = c.pages - 1                    # the nearest to any id past the pool
    c.bt[0, np.flatnonzero(c.bt[0] == last)] = c.bt[0, 6]
    c.bt[0, 6] = last
    c.upload()
    w, ages = _sums(rng, c)
    bad = c.bt.copy()
    bad[0, 6] = c.pages + 5
    c.bt_d.copy_(to_gpu(bad))
    q = _q(rng, 1, 8, 64)
    note("weighted_decode with an id outside the pool")
    out, gw, ga = _weighted(q, c, w, ages, 0, None)
    ref, tol, sums, rel = decode_ref(q, c, 0, 0)
    check(out, ref, tol)
    rw, tw, _ = _sums_ref(c, w, ages, sums, rel, 0, [99])
    rw[:, last], tw[:, last] = w[:, last], 0
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ages)


def _prompt_weights(q, c, lse, w, ages, start, window, sinks, new_keys, stream=None):
    B, R, hq, d = q.shape
    ws = workspace(kvhp.prompt_weights_workspace_bytes(B, R, hq, c.hkv, d, c.cap))
    w_d, a_d = to_gpu(w), to_gpu(ages)
    kvhp.prompt_weights(to_gpu(q), c.kv, to_gpu(lse), w_d, hq, c.hkv, d, c.cap, new_keys,
                        window=window, sinks=sinks, q_start=to_gpu(np.asarray(start, np.int32)),
                        seq_lens=c.lens_d, ages=a_d, workspace=ws, stream=stream)
    sync()
    return from_gpu(w_d), from_gpu(a_d)


def _prompt_ref(q, c, start, window, sinks):
    """lse [B][Hq][R] in fp32 and the sums over each key with their relative bound."""
    B, R, hq, d = q.shape
    G = hq // c.hkv
    lse = np.full((B, hq, R), np.nan, np.float32)   # padding rows: never read into a sum
    add, rel = {}, {}
    for b in range(B):
        n = min(int(c.lens[b]), c.cap)
        for h in range(c.hkv):
            hs = slice(h * G, (h + 1) * G)
            tot, worst = np.zeros(n), 0.0
            for r in range(R):
                p = int(start[b]) + r
                if p < 0 or p >= n:
                    continue
                see = visible(p, n, window, sinks)
                _, _, pr, ls, ds = attend(q[b, r, hs], c.k[b, h, :n], c.v[b, h, :n], see)
                lse[b, hs, r] = ls
                # the lse as rounded: an error that every weight of the row shares
                tot += (pr * np.exp(ls - lse[b, hs, r].astype(np.float64))[:, None]).sum(0)
                worst = max(worst, ds + 8 * U32 * (1 + float(np.abs(ls).max())))
            add[b, h], rel[b, h] = tot, 2 * worst + 2 * (R * G + 16) * U32
    return lse, add, rel


@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_prompt_weights_heads(hq, hkv, d):
    rng = np.random.default_rng([hq, hkv, d, 3])
    c = Cache(rng, [150, 70, 20], hkv, d).upload()
    q = _q(rng, 3, 70, hq, d)
    start = [80, 0, -50]
    w, ages = _sums(rng, c)
    for window, sinks, new in [(0, 0, 10 ** 9), (30, 4, 20)]:
        note(f"prompt_weights {hq}/{hkv} x {d} window={window}")
        lse, add, rel = _prompt_ref(q, c, start, window, sinks)
        gw, ga = _prompt_weights(q, c, lse, w, ages, start, window, sinks, new)
        rw, tw, ra = _sums_ref(c, w, ages, add, rel, new, c.lens - 1)
        _check_sums(gw, rw, tw)
        assert np.array_equal(ga, ra)


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 40), (7, 300), (32, 1000), (64, 64), (129, 129),
                                    (400, 400), (33, 2049)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 10)])
def test_prompt_weights_lengths(rows, n, window, sinks):
    rng = np.random.default_rng([rows, n])
    c = Cache(rng, [n, max(1, n // 2)], 1, 64).upload()
    q = _q(rng, 2, rows, 4, 64)
    start = [n - rows, n // 2 - rows]
    w, ages = _sums(rng, c)
    note(f"prompt_weights rows={rows} n={n} window={window}")
    lse, add, rel = _prompt_ref(q, c, start, window, sinks)
    gw, ga = _prompt_weights(q, c, lse, w, ages, start, window, sinks, n // 3)
    rw, tw, ra = _sums_ref(c, w, ages, add, rel, n // 3, c.lens - 1)
    _check_sums(gw, rw, tw)
    assert np.array_equal(ga, ra)


# ------------------------------------------------- streams, graphs, repeats --
def _calls(rng):
    """One call of each attention operator with its inputs held, and its outputs."""
    import torch
    c = Cache(rng, [900, 411, 0, 77], 2, 64).upload()
    q = to_gpu(_q(rng, 4, 8, 64))
    qp = to_gpu(_q(rng, 4, 50, 8, 64))
    start = to_gpu((c.lens - 50).astype(np.int32))
    W, S = 300, 5
    t = {"wd": torch.zeros_like(q), "od": torch.zeros_like(q), "wp": torch.zeros_like(qp),
         "lse": torch.zeros(4, 8, 50, device="cuda"),
         "w": torch.zeros(2, c.pages, PAGE, device="cuda"),
         "a": torch.zeros(2, c.pages, PAGE, dtype=torch.int32, device="cuda")}
    ws = [workspace(kvhp.window_decode_workspace_bytes(4, 8, 2, 64, 900, W, S)),
          workspace(kvhp.weighted_decode_workspace_bytes(4, 8, 2, 64, 900)),
          workspace(kvhp.window_prefill_workspace_bytes(4, 50, 8, 2, 64, 900, W, S)),
          workspace(kvhp.prompt_weights_workspace_bytes(4, 50, 8, 2, 64, 900))]

    def go(stream=None):
        kvhp.window_decode(q, c.kv, c.vv, c.lens_d, t["wd"], 8, 2, 64, 900, W, S,
                           workspace=ws[0], stream=stream)
        kvhp.window_prefill(qp, c.kv, c.vv, t["wp"], 8, 2, 64, 900, W, S, q_start=start,
                            seq_lens=c.lens_d, lse=t["lse"], workspace=ws[2], stream=stream)
        kvhp.prompt_weights(qp, c.kv, t["lse"], t["w"], 8, 2, 64, 900, 900, window=W, sinks=S,
                            q_start=start, seq_lens=c.lens_d, ages=t["a"], workspace=ws[3],
                            stream=stream)
        kvhp.weighted_decode(q, c.kv, c.vv, c.lens_d, t["od"], t["w"], 8, 2, 64, 900,
                             new_keys=0, ages=t["a"], workspace=ws[1], stream=stream)
    keep = (c, q, qp, start, ws)
    return go, t, keep


def test_streams_and_repeats_give_the_same_bits():
    import torch
    go, t, keep = _calls(np.random.default_rng(1))
    note("bounded attention: eager")
    go()
    sync()
    want = {k: x.clone() for k, x in t.items()}
    st = torch.cuda.Stream()
    for x in t.values():
        x.zero_()
    sync()
    note("bounded attention: another stream")
    go(st)
    st.synchronize()
    for k, x in t.items():
        assert torch.equal(x, want[k]), k


def test_graph_replays():
    """Captured once, replayed between eager work; every replay as the eager call."""
    import torch
    go, t, keep = _calls(np.random.default_rng(2))
    note("bounded attention: eager")
    go()
    sync()
    want = {k: x.clone() for k, x in t.items()}
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    for i in range(3):
        for x in t.values():
            x.fill_(3)
        sync()
        note(f"bounded attention: replay {i}")
        g.replay()
        sync()
        for k, x in t.items():
            live = torch.ones_like(x, dtype=torch.bool)
            if k == "wp":   # padding rows stay as they were
                live = (want[k] != 0).any(-1, keepdim=True).expand_as(x)
            if k == "lse":
                live = want[k] != 0
            if k in ("w", "a"):   # slots of no sequence stay as they were
                live = (want["w"] != 0)
            assert torch.equal(x[live], want[k][live]), k
        go()
        sync()
