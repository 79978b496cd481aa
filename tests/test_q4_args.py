"""Host checks of the appends that rotate and of the 4-bit cache's calls: the format,
what is refused, and that empty work is no work (CPU: nothing here reaches a GPU)."""
import numpy as np
import pytest

import kvhp
from q4_util import pack, quantise, unpack, values

P = 1 << 20   # stands for a device address; 16-byte aligned, never read here
BIG = 1 << 40


def _code(rc):
    return rc, kvhp.last_error()


def _append(q=P, k=P, v=P, sq=512, sk=128, sv=128, pos=P, slots=P, lens=P, theta=10000.0,
            q_out=P, pk=P, pv=P, bt=P, max_pages=64, num_pages=64, batch=2, rows=3, hq=8, hkv=2,
            d=64):
    return _code(kvhp.load().kvhp_rope_append(q, k, v, sq, sk, sv, pos, slots, lens, theta, q_out,
                                              pk, pv, bt, max_pages, num_pages, batch, rows, hq,
                                              hkv, d, None))


def _q4_append(q=P, k=P, v=P, sq=512, sk=128, sv=128, pos=P, slots=P, lens=P, theta=10000.0,
               q_out=P, pk=P, bt=P, max_pages=64, num_pages=64, batch=2, rows=3, hq=8, hkv=2,
               d=64):
    return _code(kvhp.load().kvhp_q4_rope_append(q, k, v, sq, sk, sv, pos, slots, lens, theta,
                                                 q_out, pk, bt, max_pages, num_pages, batch, rows,
                                                 hq, hkv, d, None))


def _gather(pool=P, bt=P, max_pages=64, num_pages=64, start=P, lens=P, k=P, v=P, batch=2, hkv=2,
            d=64, cap=100):
    return _code(kvhp.load().kvhp_q4_gather(pool, bt, max_pages, num_pages, start, lens, k, v,
                                            batch, hkv, d, cap, None))


def _decode(q=P, pool=P, bt=P, max_pages=64, num_pages=64, lens=P, out=P, batch=2, hq=8, hkv=2,
            d=64, cap=1000, ws=P, ws_bytes=BIG):
    return _code(kvhp.load().kvhp_q4_decode(q, pool, bt, max_pages, num_pages, lens, out, batch,
                                            hq, hkv, d, cap, ws, ws_bytes, None))


def _prefill(q=P, pool=P, bt=P, max_pages=64, num_pages=64, start=P, lens=P, out=P, lse=P,
             batch=2, rows=10, hq=8, hkv=2, d=64, cap=1000, ws=P, ws_bytes=BIG):
    return _code(kvhp.load().kvhp_q4_prefill(q, pool, bt, max_pages, num_pages, start, lens, out,
                                             lse, batch, rows, hq, hkv, d, cap, ws, ws_bytes,
                                             None))


def _refused(got, code, word):
    assert got[0] == code and word in got[1], got


INVALID, UNSUPPORTED = kvhp.KVHP_ERR_INVALID, kvhp.KVHP_ERR_UNSUPPORTED


@pytest.mark.parametrize("call", [_append, _q4_append])
def test_append_refusals(call):
    for name in ("k", "v", "bt", "pk", "q", "q_out"):   # q alone or q_out alone, too
        _refused(call(**{name: None}), INVALID, "null")
    _refused(call(max_pages=0), INVALID, "max_pages")
    _refused(call(num_pages=-1), INVALID, "num_pages")
    _refused(call(hkv=0), INVALID, "num_kv_heads")
    _refused(call(hq=0), INVALID, "num_q_heads")
    for theta in (-1.0, float("nan"), float("inf")):
        _refused(call(theta=theta), INVALID, "rope_theta")
    for d in (0, -2, 63, 258):
        _refused(call(d=d), UNSUPPORTED, "head_dim")
    _refused(call(sq=511), INVALID, "overlap")
    _refused(call(sk=127), INVALID, "overlap")
    _refused(call(sv=-128), INVALID, "overlap")
    _refused(call(batch=1 << 20, rows=1 << 20), UNSUPPORTED, "rows")
    _refused(call(hkv=65536, sk=1 << 23, sv=1 << 23), UNSUPPORTED, "KV heads")
    for empty in ({"batch": 0}, {"rows": 0}, {"batch": -1}, {"rows": -7}):
        assert call(**empty)[0] == kvhp.KVHP_OK


def test_pools():
    _refused(_append(pv=None), INVALID, "null")
    _refused(_q4_append(pk=P + 8), INVALID, "aligned")
    _refused(_q4_append(d=36, sq=288, sk=72, sv=72), UNSUPPORTED, "multiple of 8")


@pytest.mark.parametrize("call", [_gather, _decode, _prefill])
def test_cache_refusals(call):
    _refused(call(pool=None), INVALID, "null")
    _refused(call(bt=None), INVALID, "null")
    _refused(call(pool=P + 4), INVALID, "aligned")
    _refused(call(max_pages=0), INVALID, "max_pages")
    _refused(call(num_pages=0), INVALID, "num_pages")
    for d in (0, -8, 4, 100, 264):
        _refused(call(d=d), UNSUPPORTED, "head_dim")
    _refused(call(hkv=0), INVALID, "multiple")
    _refused(call(batch=65536), UNSUPPORTED, "65535")
    _refused(call(cap=(1 << 30) + 1), UNSUPPORTED, "max_seq_len")
    for empty in ({"batch": 0}, {"cap": 0}, {"batch": -1}, {"cap": -5}):
        assert call(**empty)[0] == kvhp.KVHP_OK


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_attention_refusals(call):
    _refused(call(q=None), INVALID, "null")
    _refused(call(out=None), INVALID, "null")
    _refused(call(hq=7), INVALID, "multiple")
    _refused(call(hq=-8, hkv=-2), INVALID, "multiple")
    _refused(call(hq=1 << 26, hkv=1), UNSUPPORTED, "num_q_heads")


def test_lengths_rows_and_outputs():
    _refused(_decode(lens=None), INVALID, "null")
    _refused(_gather(lens=None), INVALID, "null")
    _refused(_gather(k=None, v=None), INVALID, "null")
    _refused(_gather(k=P + 2), INVALID, "aligned")
    assert _prefill(rows=0)[0] == kvhp.KVHP_OK
    assert _prefill(rows=-3)[0] == kvhp.KVHP_OK


def test_page_bytes():
    assert [kvhp.q4_page_bytes(d) for d in (8, 64, 128, 256)] == [256, 1152, 2176, 4224]
    assert all(kvhp.q4_page_bytes(d) % 128 == 0 for d in range(8, 257, 8))
    assert all(kvhp.q4_page_bytes(d) == 0 for d in (0, -8, 4, 63, 100, 264, 1 << 30))


def test_workspaces():
    dec, pre = kvhp.q4_decode_workspace_bytes, kvhp.q4_prefill_workspace_bytes
    calls = [(_decode, dec(2, 8, 2, 64, 1000), {}), (_prefill, pre(2, 10, 8, 2, 64, 1000), {}),
             (_decode, dec(1, 32, 8, 128, 16384), {"batch": 1, "hq": 32, "hkv": 8, "d": 128,
                                                   "cap": 16384}),
             (_prefill, pre(1, 3, 32, 8, 128, 16384), {"batch": 1, "rows": 3, "hq": 32, "hkv": 8,
                                                       "d": 128, "cap": 16384})]
    for call, need, kw in calls:
        if not need:
            continue
        for ws, n in ((P, need - 1), (None, need), (P, 0)):
            _refused(call(ws=ws, ws_bytes=n, **kw), kvhp.KVHP_ERR_WORKSPACE, "workspace")
        _refused(call(ws=P + 8, ws_bytes=need, **kw), INVALID, "aligned")
    # what every call refuses has no size
    assert dec(0, 8, 2, 64, 1000) == dec(2, 7, 2, 64, 1000) == dec(2, 8, 0, 64, 1000) == 0
    assert dec(2, 8, 2, 60, 1000) == dec(2, 8, 2, 64, (1 << 30) + 1) == dec(2, 8, 2, 64, -1) == 0
    assert pre(2, 0, 8, 2, 64, 1000) == pre(2, 10, -8, 2, 64, 1000) == pre(2, 10, 8, 2, 0, 10) == 0
    assert pre(65536, 10, 8, 2, 64, 1000) == 0


def test_strides_of_the_python_calls():
    torch = pytest.importorskip("torch")
    qkv = torch.zeros((2, 3, 12, 8), dtype=torch.float16)
    rows = kvhp._token_rows
    assert rows(qkv[:, :, :8], "x") == (2, 3, 96)
    assert rows(qkv[:, :1, 8:10], "x") == (2, 1, 3 * 96)
    assert rows(qkv[:1, :1], "x") == (1, 1, 96)
    for bad in (qkv[..., ::2], qkv[:, :, ::2], qkv[:, :2], qkv.transpose(0, 1)):
        with pytest.raises(kvhp.KVHPError):
            rows(bad, "x")
    with pytest.raises(kvhp.KVHPError):
        kvhp._append_rows(qkv[:, :, :8], qkv[:1, :, 8:10], qkv[:, :, 10:], None, "x")
    with pytest.raises(kvhp.KVHPError):
        kvhp._append_rows(qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:], qkv[:, :, :8], "x")


def _rows(kind, rng, n, d):
    x = rng.standard_normal((n, d))
    return {"normal": x, "small": 1e-4 * x, "tiny": 1e-7 * x, "shifted": 100 + 0.1 * x,
            "far": -3000 + x, "large": np.clip(20000 * x, -65504, 65504),
            "heavy": x ** 5, "equal": np.repeat(x[:, :1], d, 1), "zero": 0 * x,
            "two": np.where(x > 0, 1.0, 1.0 + 2.0 ** -10), "positive": np.abs(x)}[kind]


@pytest.mark.parametrize("d", [8, 64, 128])
@pytest.mark.parametrize("kind", ["normal", "small", "tiny", "shifted", "far", "large", "heavy",
                                  "equal", "zero", "two", "positive"])
def test_format(kind, d):
    """A value is off by half of s, and by what clips at the range's ends (s/128, where r is
    rounded to 2^-6; s/2 where to 1); n + r and r - 16 are fp16 numbers."""
    rng = np.random.default_rng(d)
    x = _rows(kind, rng, 300, d).astype(np.float16)
    n, p = quantise(x)
    s, r = p[..., :1].astype(np.float64), p[..., 1:].astype(np.float64)
    codes = np.arange(16) + r
    assert np.array_equal(codes.astype(np.float16).astype(np.float64), codes)
    assert np.array_equal((r - 16).astype(np.float16).astype(np.float64), r - 16)
    assert np.isfinite(p).all() and np.abs(r).max() <= 1984
    step = 2.0 ** (np.floor(np.log2(np.abs(r) + 16)) - 10)
    x = x.astype(np.float64)
    off = np.abs(values(n, p) - x)
    assert (off <= np.abs(s) * (0.5 + 0.5 * step) * (1 + 2.0 ** -20)).all()
    spread = np.ptp(x, -1, keepdims=True) / 15
    largest = np.abs(x).max(-1, keepdims=True) / 1984
    whole = np.maximum(spread, largest)
    flat = spread == 0
    assert (flat | (s >= whole * (1 - 2.0 ** -23))).all()
    assert (flat | (s <= whole * (1 + 2.0 ** -10) + 2.0 ** -24)).all()
    assert (off[np.broadcast_to(flat, off.shape)] == 0).all()
    again = unpack(pack(n.reshape(-1, 1, 1, d).repeat(16, 2), p.reshape(-1, 1, 1, 2).repeat(16, 2),
                        n.reshape(-1, 1, 1, d).repeat(16, 2), p.reshape(-1, 1, 1, 2).repeat(16, 2)), d)
    assert np.array_equal(again[0][:, 0, 3], n) and np.array_equal(again[3][:, 0, 15], p)


def test_format_of_rows_that_are_not_finite():
    x = np.zeros((3, 8), np.float16)
    x[0, 3], x[1, 0], x[2, 7] = np.inf, -np.inf, np.nan
    n, p = quantise(x)
    assert (n == 0).all() and np.isnan(p).all() and (p.view(np.uint16) == 0x7e00).all()
