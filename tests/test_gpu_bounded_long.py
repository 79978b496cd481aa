"""Windowed prompts and chunks over caches and at sizes where a workgroup walks hundreds of
tiles of keys, against the definition in 64 bits (tolerances: bounded_util)."""
import math

import numpy as np
import pytest

import kvhp
from bounded_util import PAGE, U16, U32, check, workspace
from gpu_util import from_gpu, note, sync, to_gpu

pytestmark = pytest.mark.gpu


def _attend(q, k, v, see):
    """bounded_util.attend on the device: q [G, D], k, v [n, D] and see [n] on the GPU; the
    output and its tolerance, lse and its own."""
    import torch
    q, k, v = q.double(), k[see].double(), v[see].double()
    d, n = q.shape[1], k.shape[0]
    s = (q @ k.T.contiguous()) / math.sqrt(d)
    size = float(((q.abs() @ k.abs().T.contiguous()) / math.sqrt(d)).max())
    ds = (d + 4) * U32 * size + 4 * U32 * float(s.abs().max())
    m = s.amax(1, keepdim=True)
    e = torch.exp(s - m)
    l = e.sum(1, keepdim=True)
    p = e / l
    out = p @ v
    small = n * 2.0 ** -25 * float(v.abs().max()) / l
    tol = U16 * out.abs() + (2 * U16 + 2 * ds + 2 * n * U32) * (p @ v.abs()) + small + 2.0 ** -25
    lse = (m + l.log())[:, 0]
    return out, tol, lse, ds + (n + 8) * U32 + 4 * U32 * lse.abs()


def _see(p, n, window, sinks):
    import torch
    j = torch.arange(n, device="cuda")
    see = j <= p
    if window > 0:
        see &= (j < sinks) | (p - j < window)
    return see


def _shared(seed, B, hkv, d, n):
    """Pools of n keys in shuffled pages that every one of B sequences reads (a shared prefix),
    and the same keys in order, [Hkv][n][D]."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = (n + PAGE - 1) // PAGE
    k, v = (torch.empty((hkv, pages, PAGE, d), dtype=torch.float16, device="cuda").normal_(
        generator=g) for _ in range(2))
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    bt = to_gpu(np.tile(order, (B, 1)))
    at = to_gpu(order).long()
    return k, v, bt, [x[:, at].reshape(hkv, -1, d)[:, :n] for x in (k, v)]


@pytest.mark.parametrize("d,window,sinks", [(64, 0, 0), (64, 70001, 21), (128, 0, 0),
                                            (128, 40000, 500)])
def test_one_range_of_hundreds_of_tiles(d, window, sinks):
    """So many sequences that none is cut into ranges, over up to 140000 keys in shuffled
    pages: lengths on both sides of 256, 512, 768 and 1024 tiles of 64 keys, and a key that
    only the last row sees."""
    import torch
    B, hkv, R, n = 66, 4, 2, 140000
    k, v, bt, (kk, vv) = _shared(d, B, hkv, d, n)
    edges = [t * 64 + e for t in (256, 257, 258, 511, 512, 513, 768, 1024, 1280) for e in (-1, 0, 1, 2)]
    lens = np.array((edges + [n, 2, 3, 64, 65, 1000] + list(range(90000, 140000, 2500)))[:B], np.int32)
    lens = np.concatenate([lens, np.random.default_rng(d).integers(2, n, B - len(lens))]).astype(np.int32)
    g = torch.Generator(device="cuda").manual_seed(d + 1)
    q = torch.empty((B, R, hkv, d), dtype=torch.float16, device="cuda").normal_(generator=g)
    out, lse = torch.zeros_like(q), torch.zeros((B, hkv, R), device="cuda")
    assert kvhp.window_prefill_workspace_bytes(B, R, hkv, hkv, d, n, window, sinks) == 0
    vv = vv.clone()
    last = int(bt[0, (n - 1) // PAGE])
    v[:, last, (n - 1) % PAGE] = math.inf
    note(f"window_prefill: ranges of up to 2188 tiles, D = {d}, window {window}, {sinks} first")
    kvhp.window_prefill(q, kvhp.paged_view(k, bt), kvhp.paged_view(v, bt), out, hkv, hkv, d, n,
                        window, sinks, q_start=to_gpu(lens - R), seq_lens=to_gpu(lens), lse=lse)
    sync()
    for b in range(B):
        for r in range(R):
            p = int(lens[b]) - R + r
            see = _see(p, p + 1, window, sinks)
            for h in range(hkv):
                o, tol, ls, ltol = _attend(q[b, r, h:h + 1], kk[h, :p + 1], vv[h, :p + 1], see)
                what = f"sequence {b} of {lens[b]}, row {r}, head {h}"
                if p == n - 1:
                    assert bool((out[b, r, h] == math.inf).all()), what
                else:
                    check(from_gpu(out[b, r, h]), from_gpu(o[0]), from_gpu(tol[0]), what)
                check(from_gpu(lse[b, h, r:r + 1]), from_gpu(ls), from_gpu(ltol), what)


@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (64, 100000)])
def test_many_small_weights_beside_a_large_one(d, window):
    """One key with most of the weight and 131071 with 2^-25 of it each, 2^-8 together: their
    rounding to fp16 is an absolute 2^-25 of a reference at least 2^7 below the largest weight."""
    import torch
    B, hkv, R, n = 65, 4, 2, 131072
    k, v, bt, (kk, vv) = _shared(d, B, hkv, d, n)
    sinks = 1
    k[..., 0], v[:] = 12 - 17.35, 1.0      # 17.35 = 25.03 log 2, times the query's sqrt(D) below
    k[..., 1:] = 0
    k[:, int(bt[0, 0]), 0, 0] = 12
    v[:, int(bt[0, 0]), 0] = 0
    q = torch.zeros((B, R, hkv, d), dtype=torch.float16, device="cuda")
    q[..., 0] = math.sqrt(d)
    lens = np.linspace(n // 2, n, B).astype(np.int32)
    out = torch.zeros_like(q)
    assert kvhp.window_prefill_workspace_bytes(B, R, hkv, hkv, d, n, window, sinks) == 0
    note(f"window_prefill: many small weights, D = {d}, window {window}")
    kvhp.window_prefill(q, kvhp.paged_view(k, bt), kvhp.paged_view(v, bt), out, hkv, hkv, d, n,
                        window, sinks, q_start=to_gpu(lens - R), seq_lens=to_gpu(lens))
    sync()
    # the scores as the fp16 keys and query give them
    x = np.float64(np.float16(math.sqrt(d))) / math.sqrt(d)
    e = math.exp(x * (np.float64(np.float16(12 - 17.35)) - 12))
    got = from_gpu(out).astype(np.float64)
    for b in range(B):
        for r in range(R):
            p = int(lens[b]) - R + r
            seen = p if window == 0 else min(p, window)
            l = 1 + seen * e
            want = seen * e / l
            # relative: the output's and each weight's rounding, the scores' and the sums' in fp32
            ds = (d + 8) * U32 * 18
            tol = (3 * U16 + 2 * ds + 2 * seen * U32) * want + seen * 2.0 ** -32 / l + 2.0 ** -25
            check(got[b, r], np.full((hkv, d), want), np.full((hkv, d), tol), f"{lens[b]} keys, row {r}")


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(700, 20), (0, 0), (1500, 0)])
@pytest.mark.parametrize("paged", [False, True])
def test_long_prompts(hq, hkv, d, window, sinks, paged):
    """Prompts whose blocks of rows have their window wholly inside the text, and causal ones
    with their log-sum-exp: every row of every head."""
    import torch
    S, G = 2611, hq // hkv
    g = torch.Generator(device="cuda").manual_seed(S + d)
    if paged:
        k, v, bt, (kk, vv) = _shared(d, 1, hkv, d, S)
        views = [kvhp.paged_view(x, bt) for x in (k, v)]
    else:
        k, v = (torch.empty((1, S, hkv, d), dtype=torch.float16, device="cuda").normal_(generator=g)
                for _ in range(2))
        views = [kvhp.strided_view(x, x.stride(0), x.stride(2), x.stride(1)) for x in (k, v)]
        kk, vv = (x[0].transpose(0, 1) for x in (k, v))
    q = torch.empty((1, S, hq, d), dtype=torch.float16, device="cuda").normal_(generator=g)
    out, lse = torch.zeros_like(q), torch.zeros((1, hq, S), device="cuda")
    ws = workspace(kvhp.window_prefill_workspace_bytes(1, S, hq, hkv, d, S, window, sinks))
    note(f"window_prefill: a prompt of {S}, {hq}/{hkv} x {d}, window {window}, paged={paged}")
    kvhp.window_prefill(q, *views, out, hq, hkv, d, S, window, sinks, lse=lse, workspace=ws)
    sync()
    j = torch.arange(S, device="cuda")
    see = j[None] <= j[:, None]
    if window > 0:
        see &= (j[None] < sinks) | (j[:, None] - j[None] < window)
    for h in range(hq):
        kd, vd = kk[h // G].double(), vv[h // G].double()
        qd = q[0, :, h].double()
        s = (qd @ kd.T.contiguous()) / math.sqrt(d)
        s.masked_fill_(~see, -math.inf)
        size = ((qd.abs() @ kd.abs().T.contiguous()) / math.sqrt(d)).masked_fill_(~see, 0).amax(1)
        m = s.amax(1)
        ds = (d + 4) * U32 * size + 4 * U32 * s.masked_fill(~see, 0).abs().amax(1)
        e = torch.exp(s - m[:, None])
        l, n = e.sum(1), see.sum(1)
        p = e / l[:, None]
        want = p @ vd
        small = n * 2.0 ** -25 * vd.abs().max() / l
        tol = (U16 * want.abs() + (2 * U16 + 2 * ds + 2 * n * U32)[:, None] * (p @ vd.abs()) +
               small[:, None] + 2.0 ** -25)
        check(from_gpu(out[0, :, h]), from_gpu(want), from_gpu(tol), f"head {h}")
        want = m + l.log()
        check(from_gpu(lse[0, h]), from_gpu(want),
              from_gpu(ds + (n + 8) * U32 + 4 * U32 * want.abs()), f"lse of head {h}")
