"""Eviction plans against their definition, the moves bit by bit, and a run of
the bounded-cache operators together."""
import numpy as np
import pytest

import kvhp
from bounded_util import PAGE, Cache, attend, check, plan_ref, visible, workspace
from gpu_util import from_gpu, make_block_tables, note, sync, to_gpu

pytestmark = pytest.mark.gpu


def _plan(w, ages, bt, lens, cap, budget, sinks, recent, newest=None, fill=-7):
    import torch
    B, hkv = len(lens), w.shape[0]
    most = min(budget, max(cap - budget, 0))
    moves = torch.full((B, hkv, most, 2), fill, dtype=torch.int32, device="cuda")
    counts = torch.full((B, hkv), fill, dtype=torch.int32, device="cuda")
    new = torch.full((B,), fill, dtype=torch.int32, device="cuda")
    kvhp.evict_plan(to_gpu(w), None if ages is None else to_gpu(ages), to_gpu(bt),
                    to_gpu(np.asarray(lens, np.int32)), moves, counts, new, cap, budget, sinks,
                    recent, newest=None if newest is None else to_gpu(newest))
    sync()
    return from_gpu(moves), from_gpu(counts), from_gpu(new)


def _check_plan(w, ages, bt, lens, cap, budget, sinks, recent, newest=None):
    moves, counts, new = _plan(w, ages, bt, lens, cap, budget, sinks, recent, newest)
    for b, n in enumerate(lens):
        n = min(max(int(n), 0), cap)
        assert new[b] == min(n, budget)
        j = np.arange(n)
        for h in range(w.shape[0]):
            wj = w[h, bt[b, j // PAGE], j % PAGE]
            aj = j if ages is None else ages[h, bt[b, j // PAGE], j % PAGE]
            want = plan_ref(wj, aj, n, budget, sinks, recent,
                            n - 1 if newest is None else int(newest[b]))
            assert counts[b, h] == len(want), (b, h)
            assert [tuple(x) for x in moves[b, h, :len(want)]] == want, (b, h)
            assert (moves[b, h, len(want):] == -7).all(), (b, h)   # left as they were


def _pools(rng, lens, hkv, kind):
    bt, pages = make_block_tables(rng, lens)
    shape = (hkv, pages, PAGE)
    if kind == "spread":      # many binary orders
        w = np.exp(rng.standard_normal(shape) * 3)
    elif kind == "equal":     # ties everywhere
        w = rng.integers(0, 3, shape).astype(np.float64)
    elif kind == "near":      # keys that differ in the last bits only
        w = 1 + rng.integers(0, 50, shape) * 2.0 ** -23
    else:                     # NaN, infinities, both zeros, negative, denormal
        w = rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-42, 2.0, 3.0e38], shape)
    return bt, w.astype(np.float32)


@pytest.mark.parametrize("kind", ["spread", "equal", "near", "odd"])
@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([300, 65, 64, 63, 1, 0], 64, 4, 20), ([17, 16, 15], 16, 0, 0), ([2, 3], 1, 0, 1),
    ([1000, 513, 2000], 512, 100, 412), ([130], 129, 0, 64), ([4097, 4096], 1000, 16, 100),
    ([5000], 4999, 4, 300)])
def test_plan(kind, lens, budget, sinks, recent):
    rng = np.random.default_rng([len(lens), budget])
    bt, w = _pools(rng, lens, 2, kind)
    note(f"evict_plan {kind} lens={lens} budget={budget}")
    _check_plan(w, None, bt, lens, max(lens), budget, sinks, recent)
    # ages of a cache that was cut before: out of order, newest given
    newest = np.array([3 * n + 5 for n in lens], np.int32)
    ages = rng.integers(0, 3 * max(lens), w.shape).astype(np.int32)
    for b, n in enumerate(lens):
        j = np.arange(n)
        ages[:, bt[b, j // PAGE], j % PAGE] = rng.permutation(3 * n + 6)[:n]
    _check_plan(w, ages, bt, lens, max(lens), budget, sinks, recent, newest)


@pytest.mark.parametrize("n", [16385, 65536, 70000, 200001])
def test_plan_long(n):
    """Lengths of every thread share, past what the registers hold too."""
    rng = np.random.default_rng(n)
    bt, w = _pools(rng, [n], 1, "spread")
    note(f"evict_plan n={n}")
    _check_plan(w, None, bt, [n], n, n // 2, 4, 1000)
    bt, w = _pools(rng, [n], 1, "equal")
    _check_plan(w, None, bt, [n], n, n // 3, 0, 0)


def test_plan_capacity_and_more_protected_than_budget():
    rng = np.random.default_rng(4)
    bt, w = _pools(rng, [500], 2, "spread")
    note("evict_plan lengths above max_seq_len")
    _check_plan(w, None, bt, [500], 200, 100, 4, 10)
    # every age claims to be recent: the lowest slots stay, nothing moves
    note("evict_plan all protected")
    moves, counts, _ = _plan(w, np.full(w.shape, 900, np.int32), bt, [500], 500, 100, 0, 50,
                             np.array([900], np.int32))
    assert (counts == 0).all() and (moves == -7).all()


@pytest.mark.parametrize("d", [64, 128, 80, 33, 256, 1])
def test_apply(d):
    import torch
    rng = np.random.default_rng(d)
    lens, budget, hkv = [200, 90, 64, 300], 64, 3
    bt, w = _pools(rng, lens, hkv, "spread")
    pages = w.shape[1]
    ages = rng.integers(0, 10 ** 6, w.shape).astype(np.int32)
    k, v = (rng.standard_normal((hkv, pages, PAGE, d)).astype(np.float16) for _ in range(2))
    moves, counts, _ = _plan(w, None, bt, lens, 300, budget, 4, 16)
    bt_bad = bt.copy()
    bt_bad[3, 2] = -1                  # a destination page that is gone: its moves are dropped
    want = [x.copy() for x in (k, v, w, ages)]
    for b in range(len(lens)):
        for h in range(hkv):
            for s, t in moves[b, h, :counts[b, h]]:
                if b == 3 and t // PAGE == 2:
                    continue
                for x in want:
                    x[h, bt[b, t // PAGE], t % PAGE] = x[h, bt[b, s // PAGE], s % PAGE]
    t = [to_gpu(x) for x in (k, v, w, ages)]
    for i in range(2):                 # applying again changes nothing
        note(f"evict_apply d={d} time {i}")
        kvhp.evict_apply(*t, to_gpu(bt_bad), to_gpu(moves), to_gpu(counts))
        sync()
        for got, ref in zip(t, want):
            assert np.array_equal(from_gpu(got).view(np.uint8), ref.view(np.uint8))
    flat = torch.zeros(k.size + 1, dtype=torch.float16, device="cuda")[1:].view(k.shape)
    flat.copy_(to_gpu(k))              # unaligned pool, no sums
    note(f"evict_apply d={d} unaligned")
    kvhp.evict_apply(flat, to_gpu(v), None, None, to_gpu(bt_bad), to_gpu(moves), to_gpu(counts))
    sync()
    assert np.array_equal(from_gpu(flat).view(np.uint16), want[0].view(np.uint16))


def test_apply_more_counts_than_moves_and_slots_outside():
    rng = np.random.default_rng(1)
    bt, w = _pools(rng, [64], 1, "spread")
    k = rng.standard_normal((1, w.shape[1], PAGE, 64)).astype(np.float16)
    moves = np.array([[[[40, 3], [-1, 4], [5, -9], [10 ** 8, 6], [7, 10 ** 8]]]], np.int32)
    counts = np.array([[1000]], np.int32)
    t = [to_gpu(k), to_gpu(k), to_gpu(w)]
    note("evict_apply with slots outside")
    kvhp.evict_apply(*t, None, to_gpu(bt), to_gpu(moves), to_gpu(counts))
    sync()
    k[0, bt[0, 0], 3] = k[0, bt[0, 40 // PAGE], 40 % PAGE]
    assert np.array_equal(from_gpu(t[0]), k)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (4, 2, 128), (6, 3, 80)])
def test_a_cut_cache_served(hq, hkv, d):
    """A prompt attends with a window, its weights are summed, its cache is cut; then tokens
    are appended and attended with their weights summed, and the cache is cut again whenever
    a page is over.  Every step against the same run in 64 bits on the host."""
    import torch
    rng = np.random.default_rng([hq, hkv, d])
    B, S, G, budget, sinks, recent = 2, 150, hq // hkv, 64, 4, 24
    lens0 = np.array([S, 101], np.int32)
    cap = 160
    bt, pages = make_block_tables(rng, [cap] * B)
    W = 60
    dev = "cuda"
    qs, ks, vs = (rng.standard_normal((B, S, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    q, k, v = to_gpu(qs), to_gpu(ks), to_gpu(vs)
    pool_k = torch.full((hkv, pages, PAGE, d), float("nan"), dtype=torch.float16, device=dev)
    pool_v = torch.full_like(pool_k, float("nan"))
    w = torch.full((hkv, pages, PAGE), float("nan"), device=dev)
    ages = torch.full((hkv, pages, PAGE), -1, dtype=torch.int32, device=dev)
    bt_d, lens = to_gpu(bt), to_gpu(lens0)
    note(f"a cut cache served {hq}/{hkv} x {d}: prompt")
    # tokens past a sequence's length go to its own pages behind its keys; they are masked
    kvhp.paged_append_kv(k, v, pool_k, pool_v, bt_d, torch.zeros(B, dtype=torch.int32, device=dev),
                         B, S, hkv, d)
    kv, vv = kvhp.paged_view(pool_k, bt_d), kvhp.paged_view(pool_v, bt_d)
    out, lse = torch.zeros_like(q), torch.zeros(B, hq, S, device=dev)
    kvhp.window_prefill(q, kv, vv, out, hq, hkv, d, cap, W, sinks, seq_lens=lens, lse=lse,
                        workspace=workspace(kvhp.window_prefill_workspace_bytes(
                            B, S, hq, hkv, d, cap, W, sinks)))
    kvhp.prompt_weights(q, kv, lse, w, hq, hkv, d, cap, cap, window=W, sinks=sinks,
                        seq_lens=lens, ages=ages,
                        workspace=workspace(kvhp.prompt_weights_workspace_bytes(
                            B, S, hq, hkv, d, cap)))
    sync()
    # the host's cache: per (b, h) lists of (k, v, weight, age)
    host = {}
    for b in range(B):
        n = int(lens0[b])
        for h in range(hkv):
            hs = slice(h * G, (h + 1) * G)
            tot = np.zeros(n)
            for i in range(n):
                o, tol, p, _, _ = attend(qs[b, i, hs], ks[b, :n, h], vs[b, :n, h],
                                         visible(i, n, W, sinks))
                check(from_gpu(out[b, i, hs]), o, tol, "prompt")
                tot += p.sum(0)
            host[b, h] = [ks[b, :n, h].copy(), vs[b, :n, h].copy(), tot, np.arange(n)]
    newest = lens0 - 1
    n_now = lens0.copy()
    moves = torch.zeros(B, hkv, min(budget, cap - budget), 2, dtype=torch.int32, device=dev)
    counts = torch.zeros(B, hkv, dtype=torch.int32, device=dev)
    new_lens = torch.zeros(B, dtype=torch.int32, device=dev)
    ws = workspace(kvhp.weighted_decode_workspace_bytes(B, hq, hkv, d, cap))

    def cut():
        kvhp.evict_plan(w, ages, bt_d, lens, moves, counts, new_lens, cap, budget, sinks, recent,
                        newest=to_gpu(newest.astype(np.int32)))
        kvhp.evict_apply(pool_k, pool_v, w, ages, bt_d, moves, counts)
        sync()
        lens.copy_(new_lens)
        mv, ct = from_gpu(moves), from_gpu(counts)
        for (b, h), (hk, hv, hw, ha) in host.items():
            n = int(n_now[b])
            got = [tuple(x) for x in mv[b, h, :ct[b, h]]]
            # the device ranks its own fp32 sums: equal to the host's but for their rounding,
            # so its kept set is checked by weight, then followed
            j = np.arange(n)
            dw = from_gpu(w)[h, bt[b, j // PAGE], j % PAGE]
            for s, t in got:
                dw[t] = np.nan   # overwritten since
            assert got == sorted(got) and len(got) <= max(0, n - budget)
            stay = np.ones(n, bool)
            for s, t in got:
                stay[t] = False
            gone = [t for _, t in got] + [s for s in range(budget, n)
                                          if s not in {x for x, _ in got}]
            kept = [s for s in range(n) if s not in set(gone)]
            assert len(kept) == min(n, budget)
            safe = (ha < sinks) | (ha > newest[b] - recent)
            assert not any(safe[g] for g in gone)
            if gone:
                light = max(hw[g] for g in gone)
                for s in kept:
                    assert safe[s] or hw[s] >= light * (1 - 1e-4), (b, h, s)
            for s, t in got:
                for x in (hk, hv, hw, ha):
                    x[t] = x[s]
            host[b, h] = [x[:min(n, budget)] for x in (hk, hv, hw, ha)]
            n1 = min(n, budget)
            j = np.arange(n1)
            at = (h, bt[b, j // PAGE], j % PAGE)
            assert np.array_equal(from_gpu(pool_k)[at], host[b, h][0])
            assert np.array_equal(from_gpu(ages)[at], host[b, h][3])
            np.testing.assert_allclose(from_gpu(w)[at], host[b, h][2], rtol=1e-4)
        n_now[:] = np.minimum(n_now, budget)

    note("a cut cache served: first cut")
    cut()
    for step in range(2 * PAGE + 3):
        if (n_now >= budget + PAGE).any():
            note(f"a cut cache served: cut before step {step}")
            cut()
        qn, kn, vn = (rng.standard_normal((B, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
        kvhp.paged_append_kv(to_gpu(kn[:, None]), to_gpu(vn[:, None]), pool_k, pool_v, bt_d,
                             lens.clone(), B, 1, hkv, d)
        lens += 1
        n_now += 1
        newest = newest + 1
        o_d = torch.zeros(B, hq, d, dtype=torch.float16, device=dev)
        kvhp.weighted_decode(to_gpu(qn), kv, vv, lens, o_d, w, hq, hkv, d, cap, new_keys=1,
                             ages=ages, newest=to_gpu(newest.astype(np.int32)), workspace=ws)
        sync()
        for (b, h), x in host.items():
            hs = slice(h * G, (h + 1) * G)
            x[0] = np.concatenate([x[0], kn[b, None, h]])
            x[1] = np.concatenate([x[1], vn[b, None, h]])
            o, tol, p, _, _ = attend(qn[b, hs], x[0], x[1], np.ones(len(x[0]), bool))
            check(from_gpu(o_d[b, hs]), o, tol, f"step {step}")
            x[2] = np.concatenate([x[2], [0.0]]) + p.sum(0)
            x[3] = np.concatenate([x[3], [newest[b]]])
