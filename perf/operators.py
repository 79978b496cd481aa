"""The operators that bound a KV cache, and the attention that reads it.

Each case names a `path` and its sizes:

  window_decode   one new token per sequence attends the last `window` keys and
                  the first `sinks` ones (kvhp_window_decode).
  window_prefill  the rows of a prompt, or of a chunk behind cached keys, attend
                  the same way, row by row, and leave their log-sum-exp
                  (kvhp_window_prefill).
  weighted_decode one new token per sequence attends every key, and each cached
                  key's attention weight is added to its slot's running sum
                  (kvhp_weighted_decode).
  prompt_weights  the attention weights that the last rows of a prompt give each
                  key, added to the same sums (kvhp_prompt_weights).
  evict_plan      the slots that stay when the cache is cut to `budget` tokens,
                  per sequence and KV head: the first tokens, the most recent
                  ones, and the heaviest; and the moves that close the gaps
                  (kvhp_evict_plan).
  evict_apply     those moves, in place, in the pages (kvhp_evict_apply).

Sizes are those of the repository's configurations (32/8 heads of 64 and 128,
32/4 and 14/2 heads of 64; contexts of up to 8K for batches, 16K for one
sequence) with windows and budgets of a quarter to a half of the context.

`exact` computes the same outputs in 64 bits, row by row, from the definition.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 16
HEADS = [(32, 8, 128), (32, 8, 64), (32, 4, 64), (14, 2, 64)]


def listed():
    return [
        # the smallest call: one sequence's token, a short window, contiguous cache
        {"name": "wdecode_1x4096", "path": "window_decode", "batch": 1, "ctx": 4096, "hq": 32,
         "hkv": 8, "d": 64, "window": 1024, "sinks": 4, "paged": False},
        # batched serving: 32 ragged sequences in shuffled pages, half of the context visible
        {"name": "wdecode_32x8192", "path": "window_decode", "batch": 32, "ctx": 8192, "hq": 32,
         "hkv": 8, "d": 128, "window": 4096, "sinks": 4, "paged": True},
        # a few odd, short prompts at 7 query heads per KV head
        {"name": "wprefill_3x777", "path": "window_prefill", "batch": 3, "rows": 777, "ctx": 777,
         "hq": 14, "hkv": 2, "d": 64, "window": 200, "sinks": 5, "paged": False},
        # a long prompt
        {"name": "wprefill_8192", "path": "window_prefill", "batch": 1, "rows": 8192, "ctx": 8192,
         "hq": 32, "hkv": 8, "d": 128, "window": 2048, "sinks": 16, "paged": False},
        # a chunk of each of four prompts behind its cached keys
        {"name": "wchunk_4x128", "path": "window_prefill", "batch": 4, "rows": 128, "ctx": 8192,
         "hq": 32, "hkv": 8, "d": 128, "window": 4096, "sinks": 4, "paged": True},
        # single-sequence decoding with weights kept
        {"name": "weighted_1x2048", "path": "weighted_decode", "batch": 1, "ctx": 2048, "hq": 32,
         "hkv": 4, "d": 64},
        # batched decoding with weights kept
        {"name": "weighted_32x8192", "path": "weighted_decode", "batch": 32, "ctx": 8192,
         "hq": 32, "hkv": 8, "d": 128},
        # the last rows of odd prompts as the window that observes which keys matter
        {"name": "pweights_4x32", "path": "prompt_weights", "batch": 4, "rows": 32, "ctx": 3001,
         "hq": 32, "hkv": 4, "d": 64},
        # the weights of a whole prompt
        {"name": "pweights_4096", "path": "prompt_weights", "batch": 1, "rows": 4096,
         "ctx": 4096, "hq": 32, "hkv": 8, "d": 128},
        # one sequence cut back to its budget after a page of new tokens
        {"name": "eplan_1x2064", "path": "evict_plan", "batch": 1, "ctx": 2064, "budget": 2048,
         "hkv": 4, "sinks": 4, "recent": 256},
        # prompts of a batch cut to half of the longest
        {"name": "eplan_32x8192", "path": "evict_plan", "batch": 32, "ctx": 8192, "budget": 4096,
         "hkv": 8, "sinks": 4, "recent": 512},
        # and their rows moved
        {"name": "eapply_32x8192", "path": "evict_apply", "batch": 32, "ctx": 8192,
         "budget": 4096, "hkv": 8, "d": 128, "sinks": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    path = rng.choice(["window_decode", "window_decode", "window_prefill", "window_prefill",
                       "weighted_decode", "weighted_decode", "prompt_weights", "evict_plan",
                       "evict_apply"])
    hq, hkv, d = rng.choice(HEADS)
    batch = rng.choice([1, _log(rng, 2, 32)])
    if path in ("window_decode", "weighted_decode"):
        ctx = _log(rng, 64, 16384 if batch == 1 else 8192)
        c = {"path": path, "batch": batch, "ctx": ctx, "hq": hq, "hkv": hkv, "d": d}
        if path == "window_decode":
            c.update(window=_log(rng, 16, min(ctx, 4096)), sinks=rng.choice([0, 1, 4, 16, 37]),
                     paged=batch > 1 or rng.random() < 0.5)
        return c
    if path == "window_prefill":
        batch = rng.choice([1, 1, 2, 3, 4])
        rows = _log(rng, 2, 8192 // batch)
        behind = rng.choice([0, _log(rng, 16, 4096)])
        return {"path": path, "batch": batch, "rows": rows, "ctx": min(8192, rows + behind),
                "hq": hq, "hkv": hkv, "d": d, "window": _log(rng, 16, 2048),
                "sinks": rng.choice([0, 1, 4, 16, 37]), "paged": behind > 0}
    if path == "prompt_weights":
        batch = rng.choice([1, 1, 2, 4])
        ctx = _log(rng, 64, 4096 // batch if batch > 1 else 4096)
        return {"path": path, "batch": batch, "rows": rng.choice([ctx, _log(rng, 8, min(ctx, 256))]),
                "ctx": ctx, "hq": hq, "hkv": hkv, "d": d}
    ctx = _log(rng, 128, 16384 if batch == 1 else 8192)
    budget = max(64, int(ctx * rng.choice([0.25, 0.5, 0.9, 0.98])))
    c = {"path": path, "batch": batch, "ctx": ctx, "budget": budget, "hkv": hkv,
         "sinks": rng.choice([0, 4, 16]), "recent": _log(rng, 16, budget // 2)}
    if path == "evict_apply":
        c["d"] = d
    return c


# ---------------------------------------------------------------- inputs ----
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 1.0, generator=g)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def _lens(case, seed, least=1):
    """Lengths: the full context for one sequence; for a batch the same ragged
    lengths for every seed, in another order."""
    if case["batch"] == 1:
        return np.array([case["ctx"]], np.int32)
    rng = np.random.default_rng([case["batch"], case["ctx"]])
    lens = rng.integers(max(least, case["ctx"] // 64), case["ctx"] + 1, case["batch"])
    lens[0] = case["ctx"]
    return np.random.default_rng(seed).permutation(lens).astype(np.int32)


def _tables(lens, seed):
    """Block tables over a shuffled pool: [batch][width], -1 past each sequence; pool pages."""
    need = [(int(n) + PAGE - 1) // PAGE for n in lens]
    total = sum(need)
    perm = np.random.default_rng(seed + 1).permutation(total).astype(np.int32)
    bt = np.full((len(lens), max(need)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at:at + n]
        at += n
    return bt, total


def _cache(case, seed, s, g, paged):
    """K and V: pools in pages, or contiguous [B][Hkv][ctx][D]."""
    B, hkv, d = case["batch"], case["hkv"], case["d"]
    if paged:
        bt, pages = _tables(s["lens_h"], seed)
        s["bt"] = _dev(bt)
        shape = (hkv, pages, PAGE, d)
    else:
        shape = (B, hkv, case["ctx"], d)
    s["k"], s["v"] = _normal(g, *shape), _normal(g, *shape)


def _sums(case, seed, s, g):
    """Running weights with a heavy tail, some never attended, and the ages of a
    cache that was cut before: the newest tokens in order, the others mixed."""
    hkv, pages, ctx = case["hkv"], s["pages"], case["ctx"]
    w = torch.empty((hkv, pages, PAGE), device="cuda").exponential_(1.0, generator=g)
    s["weights"] = w.pow_(3).mul_(torch.rand(w.shape, device="cuda", generator=g) > 0.1)
    s["ages"] = torch.zeros((hkv, pages, PAGE), dtype=torch.int32, device="cuda")
    lens, B = s["lens"].long(), case["batch"]
    newest = 3 * lens
    j = torch.arange(ctx, device="cuda")
    kept = min(case.get("budget", ctx), ctx)
    order = torch.rand((hkv, B, 3 * ctx), device="cuda", generator=g).argsort(-1)[..., :ctx]
    order = case.get("sinks", 0) + order % newest[:, None]
    order = torch.where((j < case.get("sinks", 0)), j, order)
    order = torch.where((j >= kept), newest[:, None] - (lens[:, None] - 1 - j), order)
    at = _rows(s["bt"], j[None].expand(B, -1), pages)
    live = (j[None] < lens[:, None])[None].expand(hkv, -1, -1)
    flat = (torch.arange(hkv, device="cuda")[:, None, None] * (pages * PAGE) + at)[live]
    s["ages"].view(-1)[flat] = order[live].int()
    s["newest"] = newest.int()


def prepare(case, seed):
    path, B, g = case["path"], case["batch"], _gen(seed)
    s = {"path": path, "case": case}
    s["lens_h"] = lens = _lens(case, seed, least=case.get("rows", 1) if path == "window_prefill"
                               and case["paged"] else 1)
    s["lens"] = _dev(lens)
    if path in ("window_decode", "weighted_decode"):
        _cache(case, seed, s, g, path == "weighted_decode" or case["paged"])
        s["q"] = _normal(g, B, case["hq"], case["d"])
        s["out"] = torch.empty_like(s["q"])
        if path == "weighted_decode":
            s["pages"] = s["k"].shape[1]
            _sums(case, seed, s, g)
        return s
    if path == "window_prefill":
        R, hq, hkv, d = case["rows"], case["hq"], case["hkv"], case["d"]
        s["q"] = _normal(g, B, R, hq, d)
        if case["paged"]:   # the chunk's rows are each sequence's last
            _cache(case, seed, s, g, True)
            s["start"] = s["lens"] - R
        else:               # the prompts' own K/V, token by token as the projection leaves them
            s["k"], s["v"] = _normal(g, B, R, hkv, d), _normal(g, B, R, hkv, d)
            s["start"] = None
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros((B, hq, R), device="cuda")
        return s
    if path == "prompt_weights":
        R, hq = case["rows"], case["hq"]
        _cache(case, seed, s, g, True)
        s["pages"] = s["k"].shape[1]
        s["q"] = _normal(g, B, R, hq, case["d"])
        s["start"] = s["lens"] - R
        s["weights"] = torch.zeros((case["hkv"], s["pages"], PAGE), device="cuda")
        s["ages"] = torch.zeros((case["hkv"], s["pages"], PAGE), dtype=torch.int32, device="cuda")
        s["lse"] = torch.logsumexp(_scores(s, *_chunk_mask(s, 0, 0)[:2]), -1).view(B, hq, R)
        live = (s["start"][:, None] + torch.arange(R, device="cuda") >= 0)[:, None]
        s["lse"] = torch.where(live, s["lse"], 0.0)
        return s
    # eviction
    hkv, budget = case["hkv"], case["budget"]
    bt, s["pages"] = _tables(lens, seed)
    s["bt"] = _dev(bt)
    _sums(case, seed, s, g)
    s["most"] = max(1, min(budget, case["ctx"] - budget))
    s["moves"] = torch.zeros((B, hkv, s["most"], 2), dtype=torch.int32, device="cuda")
    s["counts"] = torch.zeros((B, hkv), dtype=torch.int32, device="cuda")
    s["new_lens"] = torch.zeros(B, dtype=torch.int32, device="cuda")
    if path == "evict_apply":
        _plan(s)
        s["k"] = _normal(g, hkv, s["pages"], PAGE, case["d"])
        s["v"] = _normal(g, hkv, s["pages"], PAGE, case["d"])
    return s


# ----------------------------------------------------------- plain forms ----
def _rows(bt, pos, pages):
    """Rows in a head's pool of the positions pos [B, n] through the block table."""
    page = bt.long().gather(1, (pos // PAGE).clamp(max=bt.shape[1] - 1))
    return page.clamp(0, pages - 1) * PAGE + pos % PAGE


def _take(s, name, pos):
    """K or V rows at pos [B, n] as [B, Hkv, n, D] in 32 bits."""
    x = s[name]
    if "bt" in s:
        hkv, pages, _, d = x.shape
        return x.view(hkv, pages * PAGE, d)[:, _rows(s["bt"], pos, pages)].transpose(0, 1).float()
    if s["path"] == "window_prefill":   # [B, n, Hkv, D]
        x = x.transpose(1, 2)
    at = pos.clamp(max=x.shape[2] - 1)[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])
    return x.gather(2, at).float()


def _decode(s, pos, valid):
    """softmax(q K^T / sqrt(D)) over the keys at pos [B, n]: weights [B, Hkv, G, n] and output."""
    q, hkv = s["q"], s["case"]["hkv"]
    B, hq, d = q.shape
    k, v = _take(s, "k", pos), _take(s, "v", pos)
    sc = torch.matmul(q.view(B, hkv, hq // hkv, d).float(), k.transpose(2, 3).contiguous())
    sc = (sc / math.sqrt(d)).masked_fill(~valid[:, None, None], -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    return p, torch.matmul(p, v).view(B, hq, d).half()


def _plain_window_decode(s):
    c, lens = s["case"], s["lens"].long()[:, None]
    i = torch.arange(min(c["ctx"], c["window"] + c["sinks"]), device="cuda")[None]
    low = (lens - c["window"]).clamp(min=c["sinks"])
    pos = torch.where(i < c["sinks"], i, low + i - c["sinks"])
    return _decode(s, pos, pos < lens)[1]


def _sum_index(s, n):
    """Flat indices [Hkv, B, n] of the first n positions' slots in the pools of sums."""
    hkv, B = s["case"]["hkv"], s["case"]["batch"]
    at = _rows(s["bt"], torch.arange(n, device="cuda")[None].expand(B, -1), s["pages"])
    return torch.arange(hkv, device="cuda")[:, None, None] * (s["pages"] * PAGE) + at


def _add(s, w, new_keys, newest):
    """Adds w [B, Hkv, n] to the slots' sums; the last new_keys keys start anew, with their age."""
    n = w.shape[-1]
    lens, j = s["lens"].long()[None, :, None], torch.arange(n, device="cuda")
    live = (j < lens).expand(s["case"]["hkv"], -1, -1)
    fresh = (j >= lens - new_keys).expand(s["case"]["hkv"], -1, -1)
    at = _sum_index(s, n)
    # positions past a sequence's end add nothing to a slot of its own, its first
    at = torch.where(live, at, at[..., :1])
    w = torch.where(live, w.transpose(0, 1), 0.0)
    flat = s["weights"].view(-1)
    old = torch.where(live & ~fresh, flat[at], 0.0)
    first = (old + w)[..., :1].expand_as(w)
    flat[at] = torch.where(live, old + w, first)
    ages = s["ages"].view(-1)
    age = newest[None, :, None] - (lens - 1 - j)
    age = torch.where(fresh & live, age.expand_as(at), ages[at].long())
    ages[at] = torch.where(live, age, age[..., :1].expand_as(age)).int()


def _plain_weighted_decode(s):
    n = s["case"]["ctx"]
    pos = torch.arange(n, device="cuda")[None].expand(s["case"]["batch"], -1)
    p, out = _decode(s, pos, pos < s["lens"].long()[:, None])
    _add(s, p.sum(2), 1, s["newest"].long())
    return {"out": out, "weights": s["weights"], "ages": s["ages"]}


def _chunk_mask(s, window, sinks):
    """Key positions [B, n], which of them each row sees [B, R, n], and which rows are live [B, R]."""
    c = s["case"]
    n, lens = c["ctx"], s["lens"].long()
    j = torch.arange(n, device="cuda")
    row = torch.arange(c["rows"], device="cuda")[None].expand(c["batch"], -1)
    if s["start"] is not None:
        row = row + s["start"].long()[:, None]
    see = j <= row[..., None]
    if window > 0:
        see &= (j < sinks) | (row[..., None] - j < window)
    return j[None].expand(c["batch"], -1), see, (row >= 0) & (row < lens[:, None])


def _scores(s, pos, see):
    """Masked scores [B, Hkv, G, R, n] of a chunk's rows."""
    B, R, hq, d = s["q"].shape
    hkv = s["case"]["hkv"]
    q = s["q"].view(B, R, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d).float()
    sc = torch.matmul(q, _take(s, "k", pos).transpose(2, 3).contiguous()).div_(math.sqrt(d))
    return sc.view(B, hkv, hq // hkv, R, -1).masked_fill_(~see[:, None, None], -math.inf)


def _plain_window_prefill(s):
    c = s["case"]
    pos, see, live = _chunk_mask(s, c["window"], c["sinks"])
    sc = _scores(s, pos, see)
    B, hkv, G, R, n = sc.shape
    m = sc.amax(-1, keepdim=True)
    e = sc.sub_(m).exp_()
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, hkv, G * R, n), _take(s, "v", pos)).view(B, hkv, G, R, -1) / l
    o = o.permute(0, 3, 1, 2, 4).reshape(B, R, hkv * G, -1).half()
    lse = (m + l.log()).view(B, hkv * G, R)
    return {"out": torch.where(live[:, :, None, None], o, s["out"]),
            "lse": torch.where(live[:, None], lse, s["lse"])}


def _plain_prompt_weights(s):
    pos, see, live = _chunk_mask(s, 0, 0)
    sc = _scores(s, pos, see & live[..., None])
    B, hkv, G, R, n = sc.shape
    w = sc.sub_(s["lse"].view(B, hkv, G, R, 1)).exp_().sum((2, 3))
    _add(s, w, s["case"]["ctx"], s["lens"].long() - 1)
    return {"weights": s["weights"], "ages": s["ages"]}


def _plan(s):
    """Keeps the first `budget` slots by (protected, weight, lowest slot); evicted slots below
    the budget are filled by the kept ones at or past it, both in order."""
    c = s["case"]
    n, budget, lens = c["ctx"], c["budget"], s["lens"].long()[None, :, None]
    at = _sum_index(s, n)
    j = torch.arange(n, device="cuda")
    w, age = s["weights"].view(-1)[at], s["ages"].view(-1)[at].long()
    guard = (age < c["sinks"]) | (age > s["newest"].long()[None, :, None] - c["recent"])
    live = j < lens
    rank = torch.where(live, torch.where(guard, math.inf, w), -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.zeros(rank.shape, dtype=torch.bool, device="cuda")
    keep = keep.scatter(-1, order, True) & live
    holes = (j < budget) & ~keep & (lens > budget)
    movers = (j >= budget) & keep
    counts = movers.sum(-1).transpose(0, 1)
    hkv, B, most = c["hkv"], c["batch"], s["most"]
    moves = torch.zeros((hkv, B, most + 1, 2), dtype=torch.int64, device="cuda")
    slot = j.expand(hkv, B, n)
    for_src = torch.where(movers, movers.cumsum(-1) - 1, most)
    for_dst = torch.where(holes, holes.cumsum(-1) - 1, most)
    moves[..., 0].scatter_(-1, for_src, slot)
    moves[..., 1].scatter_(-1, for_dst, slot)
    s["moves"].copy_(moves[:, :, :most].transpose(0, 1))
    s["counts"].copy_(counts)
    s["new_lens"].copy_(s["lens"].clamp(max=budget))
    return {"moves": s["moves"], "counts": s["counts"], "new_lens": s["new_lens"]}


def _plain_evict_apply(s):
    hkv, pages = s["case"]["hkv"], s["pages"]
    mv = s["moves"].long()
    live = torch.arange(s["most"], device="cuda") < s["counts"].long()[..., None]
    last = (s["lens"].long() - 1)[:, None, None]   # moved onto itself where there is no move
    src, dst = (torch.where(live, mv[..., i], last).transpose(0, 1).reshape(hkv, -1)
                for i in (0, 1))
    seq = torch.arange(s["case"]["batch"], device="cuda").repeat_interleave(s["most"])
    head = torch.arange(hkv, device="cuda")[:, None] * (pages * PAGE)
    bt = s["bt"].long()
    src, dst = (head + bt[seq, x // PAGE].clamp(0, pages - 1) * PAGE + x % PAGE
                for x in (src, dst))
    names = ("k", "v", "weights", "ages")
    flat = [s[x].view(hkv * pages * PAGE, -1) for x in names]
    flat[0][dst], flat[1][dst] = flat[0][src], flat[1][src]
    flat[2][dst], flat[3][dst] = flat[2][src], flat[3][src]
    return {x: s[x] for x in names}


# ------------------------------------------------------ the framework's calls --
def _kvhp():
    path = os.path.join(os.getcwd(), "serving-engine_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kvhp
    return kvhp


def _handles(s, kvhp):
    """The views and the workspace, which a program keeps beside its tensors."""
    c, views = s["case"], []
    for x in (s.get("k"), s.get("v")):
        if x is None:
            views.append(None)
        elif "bt" in s:
            views.append(kvhp.paged_view(x, s["bt"]))
        elif s["path"] == "window_prefill":
            views.append(kvhp.strided_view(x, x.stride(0), x.stride(2), x.stride(1)))
        else:
            views.append(kvhp.strided_view(x, x.stride(0), x.stride(1), x.stride(2)))
    need = 0
    if s["path"] == "window_decode":
        need = kvhp.window_decode_workspace_bytes(c["batch"], c["hq"], c["hkv"], c["d"], c["ctx"],
                                                  c["window"], c["sinks"])
    elif s["path"] == "weighted_decode":
        need = kvhp.weighted_decode_workspace_bytes(c["batch"], c["hq"], c["hkv"], c["d"],
                                                    c["ctx"])
    elif s["path"] == "window_prefill":
        need = kvhp.window_prefill_workspace_bytes(c["batch"], c["rows"], c["hq"], c["hkv"],
                                                   c["d"], c["ctx"], c["window"], c["sinks"])
    elif s["path"] == "prompt_weights":
        need = kvhp.prompt_weights_workspace_bytes(c["batch"], c["rows"], c["hq"], c["hkv"],
                                                   c["d"], c["ctx"])
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    s["handles"] = kvhp, views[0], views[1], ws
    return s["handles"]


def _own_run(s):
    kvhp, kv, vv, ws = s.get("handles") or _handles(s, _kvhp())
    c, path = s["case"], s["path"]
    if path == "window_decode":
        kvhp.window_decode(s["q"], kv, vv, s["lens"], s["out"], c["hq"], c["hkv"], c["d"],
                           c["ctx"], c["window"], c["sinks"], workspace=ws)
        return s["out"]
    if path == "weighted_decode":
        kvhp.weighted_decode(s["q"], kv, vv, s["lens"], s["out"], s["weights"], c["hq"], c["hkv"],
                             c["d"], c["ctx"], new_keys=1, ages=s["ages"], newest=s["newest"],
                             workspace=ws)
        return {"out": s["out"], "weights": s["weights"], "ages": s["ages"]}
    if path == "window_prefill":
        kvhp.window_prefill(s["q"], kv, vv, s["out"], c["hq"], c["hkv"], c["d"], c["ctx"],
                            c["window"], c["sinks"], q_start=s["start"], seq_lens=s["lens"],
                            lse=s["lse"], workspace=ws)
        return {"out": s["out"], "lse": s["lse"]}
    if path == "prompt_weights":
        kvhp.prompt_weights(s["q"], kv, s["lse"], s["weights"], c["hq"], c["hkv"], c["d"],
                            c["ctx"], new_keys=c["ctx"], q_start=s["start"], seq_lens=s["lens"],
                            ages=s["ages"], workspace=ws)
        return {"weights": s["weights"], "ages": s["ages"]}
    if path == "evict_plan":
        kvhp.evict_plan(s["weights"], s["ages"], s["bt"], s["lens"], s["moves"], s["counts"],
                        s["new_lens"], c["ctx"], c["budget"], c["sinks"], c["recent"],
                        newest=s["newest"])
        return {"moves": s["moves"], "counts": s["counts"], "new_lens": s["new_lens"]}
    kvhp.evict_apply(s["k"], s["v"], s["weights"], s["ages"], s["bt"], s["moves"], s["counts"])
    return {x: s[x] for x in ("k", "v", "weights", "ages")}


def run(state):
    if own:
        return _own_run(state)
    path = state["path"]
    if path == "window_decode":
        return _plain_window_decode(state)
    if path == "weighted_decode":
        return _plain_weighted_decode(state)
    if path == "window_prefill":
        return _plain_window_prefill(state)
    if path == "prompt_weights":
        return _plain_prompt_weights(state)
    return _plan(state) if path == "evict_plan" else _plain_evict_apply(state)


# ------------------------------------------------------------------ work ----
def _visible(first, rows, window, sinks):
    """Keys that the rows at positions first .. first + rows - 1 see, all together."""
    p = np.arange(max(first, 0), first + rows, dtype=np.int64)
    if window <= 0:
        return int((p + 1).sum())
    return int(np.minimum(p + 1, np.minimum(window, p + 1) + np.minimum(sinks, np.maximum(
        p + 1 - window, 0))).sum())


def work(case):
    path, B, hkv = case["path"], case["batch"], case["hkv"]
    paged_chunk = path == "window_prefill" and case["paged"]
    lens = [int(n) for n in _lens(case, 0, least=case["rows"] if paged_chunk else 1)]
    if path in ("evict_plan", "evict_apply"):
        over = [n for n in lens if n > case["budget"]]
        # about as many moves as the share of the kept slots that lies past the budget
        moves = sum(min(case["budget"], n - case["budget"]) * case["budget"] // n for n in over)
        if path == "evict_plan":
            return {"bytes": hkv * (8 * sum(over) + 8 * moves) + 8 * B, "flops": hkv * sum(over)}
        return {"bytes": hkv * max(1, moves) * (2 * (4 * case["d"] + 8) + 8), "flops": 0}
    hq, d = case["hq"], case["d"]
    if path in ("window_decode", "weighted_decode"):
        w, k = case.get("window", 0), case.get("sinks", 0)
        vis = sum(_visible(n - 1, 1, w, k) for n in lens)
        sums = 8 * hkv * vis if path == "weighted_decode" else 0
        return {"bytes": 4 * d * hkv * vis + 4 * d * hq * B + sums, "flops": 4 * d * hq * vis}
    rows = case["rows"]
    w, k = case.get("window", 0), case.get("sinks", 0)
    if path == "window_prefill":
        first = [n - rows if case["paged"] else 0 for n in lens]
        live = [min(rows, n) for n in lens]
        keys = sum(min(n, n - f if not w else min(n, n - f + w + k)) for n, f in zip(lens, first))
        vis = sum(_visible(f, r, w, k) for f, r in zip(first, live))
        return {"bytes": 4 * d * hkv * keys + (4 * d + 4) * hq * sum(live),
                "flops": 4 * d * hq * vis}
    live = [min(rows, n) for n in lens]
    vis = sum(_visible(n - rows, rows, 0, 0) for n in lens)
    return {"bytes": (2 * d + 8) * hkv * sum(lens) + (2 * d + 4) * hq * sum(live),
            "flops": 2 * d * hq * vis}


# ----------------------------------------------------------------- exact ----
def _one(s, b, h, name, n):
    """The first n rows of K or V of sequence b, KV head h, in 64 bits."""
    x = s[name]
    if "bt" in s:
        pages = s["bt"][b, :(n + PAGE - 1) // PAGE].long()
        return x[h, pages].reshape(-1, x.shape[-1])[:n].double()
    if s["path"] == "window_prefill":
        return x[b, :n, h].double()
    return x[b, h, :n].double()


def _exact_sums(s, each, new_keys):
    """The weights after each (b, h) adds each(b, h, n), a vector over the keys."""
    c = s["case"]
    w = s["weights"].double().view(c["hkv"], -1)
    for b in range(c["batch"]):
        n = int(s["lens_h"][b])
        at = torch.arange(n, device="cuda")
        row = s["bt"][b].long()[at // PAGE] * PAGE + at % PAGE
        f = max(0, n - new_keys)
        for h in range(c["hkv"]):
            add = each(b, h, n)
            w[h, row[:f]] += add[:f]
            w[h, row[f:]] = add[f:]
    return w.view(s["weights"].shape)


def exact(case, seed):
    path = case["path"]
    if path in ("evict_plan", "evict_apply"):
        return None   # whole numbers, and copies
    s = prepare(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    G = hq // hkv
    out = s["q"].double().zero_()
    if path in ("window_decode", "weighted_decode"):
        window, sinks = case.get("window", 0), case.get("sinks", 0)

        def one(b, h, n):
            sc = _one(s, b, h, "k", n) @ s["q"][b, h * G:(h + 1) * G].double().T / math.sqrt(d)
            if window > 0:
                sc[sinks:max(n - window, sinks)] = -math.inf
            p = torch.softmax(sc, 0)
            out[b, h * G:(h + 1) * G] = p.T @ _one(s, b, h, "v", n)
            return p.sum(1)
        if path == "window_decode":
            for b in range(case["batch"]):
                for h in range(hkv):
                    one(b, h, int(s["lens_h"][b]))
            return out
        return {"weights": _exact_sums(s, one, 1), "out": out, "ages": None}
    R = case["rows"]
    lse = torch.zeros((case["batch"], hq, R), dtype=torch.float64, device="cuda")

    def rows_of(b, h, n, window, sinks):
        """Live rows, and their masked scores [G, rows, n]."""
        first = 0 if s["start"] is None else n - R
        at = torch.arange(R, device="cuda") + first
        live = torch.nonzero((at >= 0) & (at < n))[:, 0]
        q = s["q"][b, live, h * G:(h + 1) * G].double().transpose(0, 1)
        sc = torch.matmul(q, _one(s, b, h, "k", n).T.contiguous()) / math.sqrt(d)
        i, j = at[live][:, None], torch.arange(n, device="cuda")[None]
        hidden = j > i
        if window > 0:
            hidden |= (j >= sinks) & (j <= i - window)
        return live, sc.masked_fill_(hidden, -math.inf)

    if path == "window_prefill":
        for b in range(case["batch"]):
            n = int(s["lens_h"][b])
            for h in range(hkv):
                live, sc = rows_of(b, h, n, case["window"], case["sinks"])
                lse[b, h * G:(h + 1) * G, live] = torch.logsumexp(sc, -1)
                o = torch.matmul(torch.softmax(sc, -1), _one(s, b, h, "v", n))
                out[b, live, h * G:(h + 1) * G] = o.transpose(0, 1)
        return {"out": out, "lse": lse}

    def add(b, h, n):
        live, sc = rows_of(b, h, n, 0, 0)
        return (sc - s["lse"][b, h * G:(h + 1) * G, live].double()[..., None]).exp().sum((0, 1))
    return {"weights": _exact_sums(s, add, case["ctx"]), "ages": None}
