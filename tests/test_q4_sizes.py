"""Sizes that the Python calls of the rotating appends and of the 4-bit cache check before
the library takes the tensors' addresses (CPU: a stand-in takes the calls)."""
import pytest

import kvhp

torch = pytest.importorskip("torch")

B, R, HQ, HKV, D, PAGES, WIDTH, T = 2, 3, 8, 2, 64, 5, 4, 10


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(kvhp, "load", lambda: lib)
    monkeypatch.setattr(kvhp, "_stream", lambda stream: None)
    return lib


def _f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _pool(h=HKV, d=D, pages=PAGES):
    return torch.zeros((h, pages, 16 * (d + 8)), dtype=torch.uint8)


def _rope(q=None, k=None, v=None, positions=None, q_out=None, pk=None, pv=None, bt=None, slots=None, lens=None,
          heads=(HQ, HKV, D)):
    x = _f16(B, R, HQ + 2 * HKV, D)
    kvhp.rope_append(x[:, :, :HQ] if q is None else q, x[:, :, HQ:HQ + HKV] if k is None else k,
                     x[:, :, HQ + HKV:] if v is None else v, positions, _f16(B, R, HQ, D) if q_out is None else q_out,
                     _f16(HKV, PAGES, 16, D) if pk is None else pk, _f16(HKV, PAGES, 16, D) if pv is None else pv,
                     _i32(B, WIDTH) if bt is None else bt, *heads, 10000.0, slots=slots, seq_lens=lens)


def _q4_rope(q=None, k=None, v=None, positions=None, q_out=None, pool=None, bt=None, slots=None, lens=None,
             heads=(HQ, HKV, D)):
    x = _f16(B, R, HQ + 2 * HKV, D)
    kvhp.q4_rope_append(x[:, :, :HQ] if q is None else q, x[:, :, HQ:HQ + HKV] if k is None else k,
                        x[:, :, HQ + HKV:] if v is None else v, positions,
                        _f16(B, R, HQ, D) if q_out is None else q_out, _pool() if pool is None else pool,
                        _i32(B, WIDTH) if bt is None else bt, *heads, 10000.0, slots=slots, seq_lens=lens)


def _gather(pool=None, bt=None, lens=None, k=None, v=None, start=None):
    kvhp.q4_gather(_pool() if pool is None else pool, _i32(B, WIDTH) if bt is None else bt,
                   _i32(B) if lens is None else lens, _f16(B, HKV, T, D) if k is None else k,
                   _f16(B, HKV, T, D) if v is None else v, start=start)


def _decode(q=None, pool=None, bt=None, lens=None, out=None, heads=(HQ, HKV, D)):
    kvhp.q4_decode(_f16(B, HQ, D) if q is None else q, _pool() if pool is None else pool,
                   _i32(B, WIDTH) if bt is None else bt, _i32(B) if lens is None else lens,
                   _f16(B, HQ, D) if out is None else out, *heads, 60)


def _prefill(q=None, pool=None, bt=None, lens=None, out=None, lse=None, start=None, heads=(HQ, HKV, D)):
    kvhp.q4_prefill(_f16(B, R, HQ, D) if q is None else q, _pool() if pool is None else pool,
                    _i32(B, WIDTH) if bt is None else bt, _f16(B, R, HQ, D) if out is None else out, *heads, 60,
                    q_start=start, seq_lens=lens, lse=lse)


GOOD = [(_rope, {}), (_rope, {"positions": _i32(B), "slots": _i32(B + 1), "lens": _i32(B)}),
        (_rope, {"bt": _i32(B + 2, WIDTH)}), (_q4_rope, {}), (_q4_rope, {"positions": _i32(B), "lens": _i32(B)}),
        (_gather, {}), (_gather, {"start": _i32(B)}), (_gather, {"bt": _i32(B + 1, WIDTH)}), (_decode, {}),
        (_decode, {"q": _f16(B, 1, HQ, D)[:, 0]}), (_prefill, {}),
        (_prefill, {"lens": _i32(B), "start": _i32(B), "lse": torch.zeros(B, HQ, R)})]

TABLES = [{"bt": _i32(B - 1, WIDTH)}, {"bt": _i32(B, 2 * WIDTH)[:, :WIDTH]}]
POOLS = [{"pool": _pool(d=128)}, {"pool": _pool(d=56)}, {"pool": _pool(h=1)},
         {"pool": _pool(pages=2 * PAGES)[:, ::2]}, {"pool": _pool(h=1).expand(HKV, -1, -1)}]
LENS = [{"lens": _i32(B - 1)}, {"lens": _i32(2 * B)[::2]}, {"lens": _i32(1).expand(B)}]
HEADS = [{"heads": h} for h in ((HQ, HKV, 128), (HQ, HKV, 32), (HQ, 4, D), (HQ, 1, D), (2 * HQ, HKV, D), (4, HKV, D))]
BAD = ([(_rope, k) for k in TABLES + LENS + HEADS +
        [{"pk": _f16(HKV, PAGES, 16, 128)}, {"pv": _f16(HKV, PAGES, 16, 32)}, {"pv": _f16(HKV, PAGES - 1, 16, D)},
         {"pk": _f16(1, PAGES, 16, D)}, {"pk": _f16(PAGES, HKV, 16, D).transpose(0, 1)}, {"positions": _i32(B - 1)},
         {"slots": _i32(2 * B)[::2]}, {"q": _f16(B, R, HQ + 1, D)}, {"k": _f16(B, R, HKV + 1, D)},
         {"v": _f16(B, R, HKV, 32)}, {"q_out": _f16(B, R, 4, D)}]] +
       [(_q4_rope, k) for k in TABLES + POOLS + LENS + HEADS +
        [{"positions": _i32(1)}, {"slots": _i32(1)}, {"q": _f16(B, R, 4, D), "q_out": _f16(B, R, 4, D)}]] +
       [(_gather, k) for k in TABLES + POOLS + LENS +
        [{"start": _i32(1)}, {"v": _f16(B, HKV, T - 1, D)}, {"k": _f16(B, T, HKV, D).transpose(1, 2)}]] +
       [(_decode, k) for k in TABLES + POOLS + HEADS +
        [{"lens": _i32(B + 1)}, {"lens": _i32(2 * B)[::2]}, {"q": _f16(B - 1, HQ, D)}, {"out": _f16(B, HQ, 32)},
         {"q": _f16(B, 2, HQ, D)[:, 0]}, {"out": _f16(HQ, B, D).transpose(0, 1)}]] +
       [(_prefill, k) for k in TABLES + POOLS + LENS + HEADS +
        [{"start": _i32(1)}, {"lse": torch.zeros(B, R)}, {"lse": torch.zeros(B, R, HQ).transpose(1, 2)},
         {"out": _f16(B, R - 1, HQ, D)}, {"q": _f16(B, R + 1, HQ, D)[:, 1:]}]])


@pytest.mark.parametrize("call,kw", GOOD)
def test_calls_that_fit(library, call, kw):
    call(**kw)
    assert len(library.calls) == 1


@pytest.mark.parametrize("call,kw", BAD)
def test_sizes_that_do_not_fit(library, call, kw):
    with pytest.raises(kvhp.KVHPError) as e:
        call(**kw)
    assert e.value.code == kvhp.KVHP_ERR_INVALID and not library.calls
