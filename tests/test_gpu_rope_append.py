"""The appends that rotate on the way: q and K against the rotation in 64 bits, V and
what must not change bit for bit, and 4-bit pages bit for bit against the format's
definition of the same fp16 rows."""
import numpy as np
import pytest

import kvhp
from gpu_util import from_gpu, note, sync, to_gpu
from q4_util import PAGE, U16, check, quantise, rotated, unpack, values

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

THETA = 10000.0
FILL = 0x5a   # what the pools hold before


class Case:
    """Rows of B sequences as parts of one fused projection, tables over a shuffled
    pool, and pools of either kind that are full of one byte."""

    def __init__(self, seed, B, R, hq, hkv, d, start, cut=0, lens=None, scale=1.0):
        rng = np.random.default_rng(seed)
        self.B, self.R, self.hq, self.hkv, self.d = B, R, hq, hkv, d
        self.slots = np.broadcast_to(np.asarray(start, np.int32), (B,)).copy()
        self.pos = (self.slots + np.asarray(cut)).astype(np.int32)
        self.lens = None if lens is None else np.asarray(lens, np.int32)
        need = max(1, (int(self.slots.max()) + R + PAGE - 1) // PAGE)
        self.pages = B * need + 3
        self.bt = rng.permutation(self.pages)[:B * need].reshape(B, need).astype(np.int32)
        self.x = (rng.standard_normal((B, R, hq + 2 * hkv, d)) * scale).astype(np.float16)

    def rows(self):
        """(b, r, page, row in it) of the rows that are written."""
        out = []
        for b in range(self.B):
            for r in range(self.R):
                s = int(self.slots[b]) + r
                if s < 0 or (self.lens is not None and s >= self.lens[b]):
                    continue
                pid = self.bt[b, s // PAGE] if s // PAGE < self.bt.shape[1] else -1
                out.append((b, r, pid if 0 <= pid < self.pages else -1, s % PAGE))
        return out

    def tensors(self, fused=True):
        x = to_gpu(self.x)
        parts = x[:, :, :self.hq], x[:, :, self.hq:self.hq + self.hkv], x[:, :, self.hq + self.hkv:]
        return parts if fused else tuple(t.contiguous() for t in parts)

    def run(self, q4, theta=THETA, fused=True, slots=True, alias=False, with_q=True):
        q, k, v = self.tensors(fused)
        dev = lambda a: None if a is None else to_gpu(a)   # noqa: E731
        if alias:
            q_out = q = q.contiguous()
        else:
            q_out = torch.full((self.B, self.R, self.hq, self.d), 7.0, dtype=torch.float16,
                               device="cuda")
        if not with_q:
            q = q_out = None
        args = (self.hq, self.hkv, self.d, theta)
        kw = {"slots": dev(self.slots) if slots else None, "seq_lens": dev(self.lens)}
        if q4:
            pool = torch.full((self.hkv, self.pages, kvhp.q4_page_bytes(self.d)), FILL,
                              dtype=torch.uint8, device="cuda")
            kvhp.q4_rope_append(q, k, v, to_gpu(self.pos), q_out, pool, to_gpu(self.bt), *args, **kw)
            pools = from_gpu(pool)
        else:
            pools = [torch.full((self.hkv, self.pages, PAGE, 2 * self.d), FILL, dtype=torch.uint8,
                                device="cuda").view(torch.float16) for _ in range(2)]
            kvhp.rope_append(q, k, v, to_gpu(self.pos), q_out, *pools, to_gpu(self.bt), *args, **kw)
            pools = [from_gpu(p) for p in pools]
        sync()
        return None if q_out is None else from_gpu(q_out), pools

    def check(self, theta=THETA, **kw):
        """Both kinds of pages."""
        note(f"append B={self.B} R={self.R} {self.hq}/{self.hkv}x{self.d} theta={theta} {kw}")
        q, (pk, pv) = self.run(False, theta, **kw)
        old = np.full((self.B, self.R, self.hq, self.d), 7.0, np.float16)
        if kw.get("alias"):
            old = self.x[:, :, :self.hq]
        rows = self.rows()
        written = np.zeros((self.pages, PAGE), bool)
        live = np.zeros((self.B, self.R), bool)
        want_k = np.full(pk.shape, FILL * 0x101, np.uint16).view(np.float16)
        want_v = want_k.copy()
        for b, r, pid, o in rows:
            live[b, r] = True
            if pid < 0:
                continue
            written[pid, o] = True
            y, e = rotated(self.x[b, r, self.hq:self.hq + self.hkv], int(self.pos[b]) + r, theta)
            check(pk[:, pid, o], y, U16 * np.abs(y) + e + 2.0 ** -25, f"K of {b}, {r}")
            want_k[:, pid, o] = pk[:, pid, o]
            want_v[:, pid, o] = self.x[b, r, self.hq + self.hkv:]
        assert np.array_equal(pk.view(np.uint16), want_k.view(np.uint16)), "K beside the rows"
        assert np.array_equal(pv.view(np.uint16), want_v.view(np.uint16)), "V"
        if q is not None:
            at = self.pos[:, None].astype(np.int64) + np.arange(self.R)
            y, e = rotated(self.x[:, :, :self.hq], np.broadcast_to(at[..., None], q.shape[:3]), theta)
            check(q[live], y[live], (U16 * np.abs(y) + e + 2.0 ** -25)[live], "q")
            assert np.array_equal(q[~live], old[~live])
        # 4 bits: the same fp16 rows' codes, and every other byte as it was
        q2, pool = self.run(True, theta, **kw)
        if q is not None:
            assert np.array_equal(q.view(np.uint16), q2.view(np.uint16))
        got = unpack(pool, self.d)
        kn, kp = quantise(pk)
        vn, vp = quantise(pv)
        fill = unpack(np.full_like(pool, FILL), self.d)
        for g, w, f, name in zip(got, (kn, kp, vn, vp), fill, ("K codes", "K numbers", "V codes",
                                                              "V numbers")):
            w = np.where(written[None, :, :, None], w, f)
            kind = np.uint16 if g.dtype == np.float16 else np.uint8
            assert np.array_equal(np.ascontiguousarray(g).view(kind), np.ascontiguousarray(w).view(kind)), name


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (32, 4, 64), (14, 2, 64), (4, 4, 64), (3, 1, 128),
                                      (8, 2, 96), (5, 1, 256), (2, 2, 8), (6, 3, 40), (4, 2, 80)])
@pytest.mark.parametrize("B,R", [(1, 1), (3, 1), (2, 17), (1, 50)])
def test_heads_and_rows(hq, hkv, d, B, R):
    Case(hq + d + R, B, R, hq, hkv, d, start=np.arange(B) * 7 + 5, cut=100).check()


@pytest.mark.parametrize("R", [1, 2, 15, 16, 31, 33, 100])
@pytest.mark.parametrize("start", [0, 1, 15, 16, 4095])
def test_slots(R, start):
    Case(R + start, 2, R, 14, 2, 64, start=[start, max(0, start - 3)], cut=[0, 1000]).check()


def test_separate_tensors_no_slots_and_theta():
    Case(1, 2, 21, 8, 2, 128, start=[30, 3]).check(fused=False, slots=False)
    Case(2, 2, 21, 8, 2, 64, start=[30, 3]).check(theta=500000.0)
    Case(3, 2, 21, 8, 2, 64, start=[30, 3]).check(theta=0.0)
    Case(4, 2, 21, 8, 2, 64, start=[30, 3]).check(theta=0.5)
    Case(5, 3, 5, 8, 2, 128, start=0).check(with_q=False)
    Case(6, 3, 5, 8, 2, 64, start=0).check(alias=True)
    Case(7, 1, 40, 8, 2, 128, start=0).check(alias=True, fused=False)


@pytest.mark.parametrize("d", [64, 128, 24])
def test_padding(d):
    """Rows before the sequence, at and past its end: neither read nor written."""
    c = Case(d, 5, 20, 6, 2, d, start=[-20, -19, -4, 0, 7], cut=3, lens=[20, 1, 9, 0, 13])
    for b in range(c.B):
        for r in range(c.R):
            s = int(c.slots[b]) + r
            if s < 0 or s >= c.lens[b]:
                c.x[b, r] = np.nan
    c.check()
    c = Case(d + 1, 3, 40, 6, 2, d, start=[-40, -25, -39])
    c.check()


@pytest.mark.parametrize("d", [64, 128, 24])
def test_dropped_pages(d):
    """Page ids outside the pool, and slots past the table, drop K and V but not q."""
    c = Case(d, 3, 40, 6, 2, d, start=[0, 5, 16])
    c.bt[0, 1], c.bt[1, 0], c.bt[2, 1], c.bt[2, 2] = -1, c.pages, 1 << 30, -(1 << 31)
    c.check()
    c = Case(d + 1, 2, 40, 6, 2, d, start=[0, 5])
    c.bt = np.ascontiguousarray(c.bt[:, :2])
    c.check()


@pytest.mark.parametrize("d", [64, 128, 24])
def test_far_positions(d):
    """fp16 accuracy at any position: the angle is no fp32 number."""
    big = (1 << 31) - 1
    c = Case(d, 6, 3, 4, 2, d, start=[0, 40, 7, 1, 2, 3])
    c.pos = np.array([8191, 131072, 1 << 24, big - 1, -1, -big], np.int32)
    c.check()


@pytest.mark.parametrize("d", [64, 128, 24])
def test_values(d):
    """Rows of every kind: equal values, far from 0, at fp16's limits, not finite."""
    c = Case(d, 2, 24, 4, 2, d, start=3)
    x = c.x[:, :, 4:].astype(np.float64)   # K and V
    kinds = [lambda y: 1e-4 * y, lambda y: 1e-7 * y, lambda y: 100 + 0.1 * y, lambda y: -3000 + y,
             lambda y: np.clip(20000 * y, -65504, 65504), lambda y: y ** 5, lambda y: 0 * y,
             lambda y: np.repeat(y[..., :1], d, -1), lambda y: np.abs(y),
             lambda y: np.where(y > 0, 65504, -65504), lambda y: np.where(y > 0, 1, 1 + 2.0 ** -10)]
    for r in range(c.R - 3):
        x[:, r] = kinds[r % len(kinds)](x[:, r])
    with np.errstate(over="ignore"):
        c.x[:, :, 4:] = x.astype(np.float16)
    c.check(theta=0.0)
    c.x[0, 21, 4, 5], c.x[0, 22, 7, d - 1], c.x[1, 23, 6, 0] = np.inf, np.nan, -np.inf
    c.x[1, 2, 5, d // 2], c.x[1, 3, 4, 1] = -np.inf, np.nan
    note(f"append rows that are not finite d={d}")
    _, pool = c.run(True, theta=0.0)
    _, (pk, pv) = c.run(False, theta=0.0)
    got = unpack(pool, d)
    rows = [(p, o) for _, _, p, o in c.rows()]
    page, row = np.array(rows).T
    for i, src in ((0, pk), (2, pv)):
        n, p = quantise(src[:, page, row])
        assert np.array_equal(got[i][:, page, row], n)
        assert np.array_equal(got[i + 1][:, page, row].view(np.uint16), p.view(np.uint16))


@pytest.mark.parametrize("hkv,d", [(2, 64), (8, 128), (3, 24)])
def test_gather(hkv, d):
    """Rows read back from any position, zeros outside the sequence."""
    c = Case(d, 3, 70, 4, hkv, d, start=[0, 9, 2])
    q, k, v = c.tensors()
    pool = torch.full((hkv, c.pages, kvhp.q4_page_bytes(d)), FILL, dtype=torch.uint8, device="cuda")
    kvhp.q4_rope_append(None, k, v, to_gpu(c.pos), None, pool, to_gpu(c.bt), 0, hkv, d, 0.0,
                        slots=to_gpu(c.slots))
    lens = c.slots + 70 - np.array([0, 5, 33], np.int32)
    start = np.array([-3, 9, 16], np.int32)
    parts = unpack(from_gpu(pool), d)
    kx, vx = values(*parts[:2]), values(*parts[2:])
    for st, n in ((start, 41), (None, 90), (start, 1)):
        ok = torch.full((3, hkv, n, d), 7.0, dtype=torch.float16, device="cuda")
        ov = ok.clone()
        note(f"q4_gather {hkv} x {d} start={st} n={n}")
        kvhp.q4_gather(pool, to_gpu(c.bt), to_gpu(lens), ok, ov, start=None if st is None else to_gpu(st))
        only = ok.clone()
        kvhp.q4_gather(pool, to_gpu(c.bt), to_gpu(lens), None, only, start=None if st is None else to_gpu(st))
        sync()
        assert torch.equal(only, ov)
        for b in range(3):
            at = (0 if st is None else int(st[b])) + np.arange(n)
            inside = (at >= 0) & (at < lens[b])
            j = np.where(inside, at, 0)
            page = c.bt[b, j // PAGE]
            for got, x in ((ok, kx), (ov, vx)):
                # codes and numbers give 15 bits and more: one rounding, or an fp32 one before it
                want = np.where(inside[None, :, None], x[:, page, j % PAGE], 0.0)
                check(from_gpu(got)[b], want, np.abs(want) * (U16 + 2.0 ** -24) + 2.0 ** -25)


def test_other_stream_graph_and_decode_rows():
    """32 new tokens on another stream, and replayed from a graph over other inputs."""
    c = Case(9, 32, 1, 32, 8, 128, start=np.arange(32) * 5)
    want_q, want = c.run(True)
    q, k, v = (t.clone() for t in c.tensors(fused=False))
    pos, slots, bt = to_gpu(c.pos), to_gpu(c.slots), to_gpu(c.bt)
    pool = torch.full((8, c.pages, kvhp.q4_page_bytes(128)), FILL, dtype=torch.uint8, device="cuda")
    q_out = torch.zeros_like(q)
    note("append on another stream")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kvhp.q4_rope_append(q, k, v, pos, q_out, pool, bt, 32, 8, 128, THETA, slots=slots, stream=side)
    side.synchronize()
    assert np.array_equal(from_gpu(pool), want) and np.array_equal(from_gpu(q_out), want_q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kvhp.q4_rope_append(q, k, v, pos, q_out, pool, bt, 32, 8, 128, THETA, slots=slots)
    src = [q.clone(), k.clone(), v.clone()]
    for i in range(4):
        note(f"append: replay {i}")
        for t, s in zip((q, k, v), src):
            t.copy_(s * (i + 1))
        pool.fill_(FILL)
        graph.replay()
        sync()
        eager, eq = torch.full_like(pool, FILL), torch.zeros_like(q)
        kvhp.q4_rope_append(q, k, v, pos, eq, eager, bt, 32, 8, 128, THETA, slots=slots)
        sync()
        assert torch.equal(pool, eager) and torch.equal(q_out, eq)


def test_odd_alignments():
    """Tensors that begin at an odd half."""
    c = Case(11, 2, 9, 6, 2, 64, start=[4, 0])
    want_q, want = c.run(True)
    flat = torch.zeros(c.x.size + 1, dtype=torch.float16, device="cuda")
    flat[1:] = to_gpu(c.x).flatten()
    x = flat[1:].view(c.x.shape)
    pool = torch.full((2, c.pages, kvhp.q4_page_bytes(64)), FILL, dtype=torch.uint8, device="cuda")
    q_out = torch.full((2 * 9 * 6 * 64 + 1,), 7.0, dtype=torch.float16, device="cuda")[1:].view(2, 9, 6, 64)
    note("append off 16-byte alignment")
    kvhp.q4_rope_append(x[:, :, :6], x[:, :, 6:8], x[:, :, 8:], to_gpu(c.pos), q_out, pool,
                        to_gpu(c.bt), 6, 2, 64, THETA, slots=to_gpu(c.slots))
    sync()
    assert np.array_equal(from_gpu(pool), want) and np.array_equal(from_gpu(q_out), want_q)
