"""Host checks of the bounded-cache operators: what they refuse, and that empty
work is no work (CPU: nothing here reaches a GPU)."""
import ctypes

import pytest

import kvhp

P = 1 << 20   # stands for a device address; 16-byte aligned, never read here


def _view(paged=True, data=P, **kw):
    v = kvhp.KVView()
    v.data, v.stride_b, v.stride_h, v.stride_s, v.stride_d = data, 0, 64 * 1024, 64, 1
    v.block_table = P if paged else None
    v.max_pages, v.page_size, v.num_pages = 64, 16, 64
    for name, x in kw.items():
        setattr(v, name, x)
    return v


def _code(rc):
    return rc, kvhp.last_error()


def _wd(q=P, k=None, v=None, lens=P, out=P, batch=2, hq=8, hkv=2, d=64, cap=1000, window=100,
        sinks=4, ws=P, ws_bytes=1 << 40):
    k, v = (x if x is not None else _view() for x in (k, v))
    return _code(kvhp.load().kvhp_window_decode(
        q, ctypes.byref(k) if k else None, ctypes.byref(v) if v else None, lens, out, batch, hq,
        hkv, d, cap, window, sinks, ws, ws_bytes, None))


def _wp(q=P, k=None, v=None, start=P, lens=P, out=P, lse=P, batch=2, rows=10, hq=8, hkv=2, d=64,
        cap=1000, window=100, sinks=4, ws=P, ws_bytes=1 << 40):
    k, v = (x if x is not None else _view() for x in (k, v))
    return _code(kvhp.load().kvhp_window_prefill(
        q, ctypes.byref(k) if k else None, ctypes.byref(v) if v else None, start, lens, out, lse,
        batch, rows, hq, hkv, d, cap, window, sinks, ws, ws_bytes, None))


def _sd(q=P, k=None, v=None, lens=P, out=P, w=P, ages=P, batch=2, hq=8, hkv=2, d=64, cap=1000,
        new_keys=1, ws=P, ws_bytes=1 << 40):
    k, v = (x if x is not None else _view() for x in (k, v))
    return _code(kvhp.load().kvhp_weighted_decode(
        q, ctypes.byref(k), ctypes.byref(v), lens, None, out, w, ages, batch, hq, hkv, d, cap,
        new_keys, ws, ws_bytes, None))


def _pw(q=P, k=None, lse=P, w=P, ages=P, batch=2, rows=10, hq=8, hkv=2, d=64, cap=1000, window=0,
        sinks=0, new_keys=1, ws=P, ws_bytes=1 << 40):
    k = k if k is not None else _view()
    return _code(kvhp.load().kvhp_prompt_weights(
        q, ctypes.byref(k), lse, None, None, None, w, ages, batch, rows, hq, hkv, d, cap, window,
        sinks, new_keys, ws, ws_bytes, None))


def _plan(w=P, ages=P, bt=P, max_pages=64, lens=P, moves=P, counts=P, new=2 * P, batch=2, hkv=2,
          pages=64, cap=1000, budget=500, sinks=4, recent=100, most=500):
    return _code(kvhp.load().kvhp_evict_plan(w, ages, bt, max_pages, lens, None, moves, counts,
                                             new, batch, hkv, pages, cap, budget, sinks, recent,
                                             most, None))


def _apply(k=P, v=P, bt=P, max_pages=64, moves=P, counts=P, batch=2, hkv=2, d=64, pages=64,
           most=10):
    return _code(kvhp.load().kvhp_evict_apply(k, v, None, None, bt, max_pages, moves, counts,
                                              batch, hkv, d, pages, most, None))


ATTENTION = [_wd, _wp, _sd, _pw]


def _refused(got, code, word):
    assert got[0] == code and word in got[1], got


@pytest.mark.parametrize("call", ATTENTION)
def test_attention_shapes(call):
    _refused(call(q=None), kvhp.KVHP_ERR_INVALID, "null")
    _refused(call(hq=7), kvhp.KVHP_ERR_INVALID, "multiple")
    _refused(call(hkv=0), kvhp.KVHP_ERR_INVALID, "multiple")
    _refused(call(hq=-8, hkv=-2), kvhp.KVHP_ERR_INVALID, "multiple")
    _refused(call(d=0), kvhp.KVHP_ERR_UNSUPPORTED, "head_dim")
    _refused(call(d=257), kvhp.KVHP_ERR_UNSUPPORTED, "head_dim")
    _refused(call(batch=65536), kvhp.KVHP_ERR_UNSUPPORTED, "65535")
    _refused(call(cap=(1 << 30) + 1), kvhp.KVHP_ERR_UNSUPPORTED, "max_seq_len")
    _refused(call(k=_view(data=None)), kvhp.KVHP_ERR_INVALID, "K view")
    _refused(call(k=_view(page_size=32)), kvhp.KVHP_ERR_INVALID, "K paged view")
    _refused(call(k=_view(num_pages=0)), kvhp.KVHP_ERR_INVALID, "K paged view")
    for empty in ({"batch": 0}, {"cap": 0}, {"batch": -1}, {"cap": -5}):
        assert call(**empty)[0] == kvhp.KVHP_OK


@pytest.mark.parametrize("call", [_wd, _wp, _sd])
def test_views(call):
    _refused(call(v=_view(data=None)), kvhp.KVHP_ERR_INVALID, "V view")
    _refused(call(v=_view(False)), kvhp.KVHP_ERR_INVALID, "both")
    _refused(call(out=None), kvhp.KVHP_ERR_INVALID, "null")


@pytest.mark.parametrize("call", [_wd, _wp, _pw])
def test_window_arguments(call):
    _refused(call(window=-1), kvhp.KVHP_ERR_INVALID, "window")
    _refused(call(sinks=-1), kvhp.KVHP_ERR_INVALID, "sinks")


@pytest.mark.parametrize("call", [_sd, _pw])
def test_sums_arguments(call):
    _refused(call(w=None), kvhp.KVHP_ERR_INVALID, "weights")
    _refused(call(new_keys=-1), kvhp.KVHP_ERR_INVALID, "new_keys")
    _refused(call(w=P + 4), kvhp.KVHP_ERR_INVALID, "aligned")
    _refused(call(ages=P + 8), kvhp.KVHP_ERR_INVALID, "aligned")
    kw = {"k": _view(False)} if call is _pw else {"k": _view(False), "v": _view(False)}
    _refused(call(**kw), kvhp.KVHP_ERR_UNSUPPORTED, "paged")


def test_lengths_and_rows():
    _refused(_wd(lens=None), kvhp.KVHP_ERR_INVALID, "null")
    _refused(_sd(lens=None), kvhp.KVHP_ERR_INVALID, "null")
    _refused(_pw(lse=None), kvhp.KVHP_ERR_INVALID, "null")
    assert _wp(rows=0)[0] == kvhp.KVHP_OK and _pw(rows=-1)[0] == kvhp.KVHP_OK


def test_workspaces():
    """Too small, absent or unaligned where one is needed."""
    lib = kvhp.load()
    need = lib.kvhp_weighted_decode_workspace_bytes(2, 8, 2, 64, 1000)
    assert need > 0
    _refused(_sd(ws_bytes=need - 1), kvhp.KVHP_ERR_WORKSPACE, "needed")
    _refused(_sd(ws=None), kvhp.KVHP_ERR_WORKSPACE, "needed")
    _refused(_sd(ws=P + 8, ws_bytes=need), kvhp.KVHP_ERR_INVALID, "aligned")
    for call, n in ((_wd, lib.kvhp_window_decode_workspace_bytes(2, 8, 2, 64, 1000, 100, 4)),
                    (_wp, lib.kvhp_window_prefill_workspace_bytes(2, 10, 8, 2, 64, 1000, 100, 4)),
                    (_pw, lib.kvhp_prompt_weights_workspace_bytes(2, 10, 8, 2, 64, 1000))):
        if n:
            _refused(call(ws_bytes=n - 1), kvhp.KVHP_ERR_WORKSPACE, "needed")
    assert lib.kvhp_window_decode_workspace_bytes(0, 8, 2, 64, 1000, 100, 4) == 0
    assert lib.kvhp_weighted_decode_workspace_bytes(2, 8, 2, 64, 0) == 0
    assert lib.kvhp_prompt_weights_workspace_bytes(2, 0, 8, 2, 64, 1000) == 0
    assert lib.kvhp_window_prefill_workspace_bytes(2, 10, -8, 2, 64, 1000, 100, 4) == 0


def test_plan_arguments():
    for name in ("w", "bt", "lens", "counts", "new", "moves"):
        _refused(_plan(**{name: None}), kvhp.KVHP_ERR_INVALID,
                 "room" if name == "moves" else "null")
    for kw in ({"hkv": 0}, {"max_pages": 0}, {"pages": -1}):
        _refused(_plan(**kw), kvhp.KVHP_ERR_INVALID, "positive")
    for kw in ({"budget": 0}, {"budget": 103}, {"sinks": -1}, {"recent": -1},
               {"sinks": 2 ** 31 - 1, "recent": 2 ** 31 - 1}):
        _refused(_plan(**kw), kvhp.KVHP_ERR_INVALID, "budget")
    _refused(_plan(most=499), kvhp.KVHP_ERR_INVALID, "room")
    _refused(_plan(new=P), kvhp.KVHP_ERR_INVALID, "alias")
    _refused(_plan(w=P + 4), kvhp.KVHP_ERR_INVALID, "aligned")
    _refused(_plan(batch=65536), kvhp.KVHP_ERR_UNSUPPORTED, "65535")
    _refused(_plan(cap=2 ** 31 - 1), kvhp.KVHP_ERR_UNSUPPORTED, "max_seq_len")
    assert _plan(batch=0)[0] == kvhp.KVHP_OK


def test_apply_arguments():
    for name in ("k", "v", "bt", "moves", "counts"):
        _refused(_apply(**{name: None}), kvhp.KVHP_ERR_INVALID, "null")
    _refused(_apply(hkv=0), kvhp.KVHP_ERR_INVALID, "positive")
    _refused(_apply(moves=P + 4), kvhp.KVHP_ERR_INVALID, "aligned")
    _refused(_apply(d=300), kvhp.KVHP_ERR_UNSUPPORTED, "head_dim")
    _refused(_apply(batch=65536), kvhp.KVHP_ERR_UNSUPPORTED, "65535")
    assert _apply(most=0)[0] == kvhp.KVHP_OK and _apply(batch=0)[0] == kvhp.KVHP_OK


def test_sizes_that_no_call_has():
    """Counts whose products leave 32 bits: refused, and their workspaces are nothing."""
    lib = kvhp.load()
    _refused(_apply(most=2 ** 31 - 1), kvhp.KVHP_ERR_UNSUPPORTED, "max_moves")
    assert lib.kvhp_weighted_decode_workspace_bytes(2, 8, 2, 64, 2 ** 31 - 1) <= 2 * 8 * 4
    assert lib.kvhp_window_decode_workspace_bytes(2, 8, 2, 64, 2 ** 31 - 1, 0, 0) == 0


@pytest.mark.parametrize("window,sinks", [(1, -1), (5, -10), (-1, 0), (-5, 3), (0, -1), (-1, -1),
                                          (-2 ** 31, -2 ** 31)])
def test_size_queries_of_refused_windows(window, sinks):
    """The size is asked before the call that refuses these: none is needed."""
    lib = kvhp.load()
    for d in (64, 128):
        assert lib.kvhp_window_decode_workspace_bytes(1, 8, 2, d, 1000, window, sinks) == 0
        assert lib.kvhp_window_prefill_workspace_bytes(1, 10, 8, 2, d, 1000, window, sinks) == 0


@pytest.mark.parametrize("batch,rows,hq,hkv,cap", [
    (1 << 30, 1 << 30, 1 << 30, 1, 1000), (1 << 20, 1 << 30, 1 << 30, 1 << 14, 1000),
    (1 << 30, 64, 1 << 30, 1 << 30, 1 << 30), (65536, 10, 8, 2, 1000), (1, 10, 1 << 26, 1, 1000),
    (1, 2 ** 31 - 1, 2 ** 31 - 1, 1, 2 ** 31 - 1), (1, 1 << 30, 1, 1, (1 << 30) + 1)])
def test_size_queries_of_refused_counts(batch, rows, hq, hkv, cap):
    """Counts whose products leave 64 bits, and others that no call takes."""
    lib = kvhp.load()
    assert lib.kvhp_window_decode_workspace_bytes(batch, hq, hkv, 64, cap, 5, 3) == 0
    assert lib.kvhp_window_prefill_workspace_bytes(batch, rows, hq, hkv, 64, cap, 5, 3) == 0
    assert lib.kvhp_prompt_weights_workspace_bytes(batch, rows, hq, hkv, 64, cap) == 0


@pytest.mark.parametrize("call", ATTENTION)
def test_more_heads_than_a_grid_has(call):
    _refused(call(hq=1 << 26, hkv=1), kvhp.KVHP_ERR_UNSUPPORTED, "num_q_heads")


def test_more_rows_than_a_grid_has():
    _refused(_wp(rows=1 << 30), kvhp.KVHP_ERR_UNSUPPORTED, "rows")


def test_null_views():
    lib, view = kvhp.load(), ctypes.byref(_view())
    for k, v, name in ((None, view, "K view"), (view, None, "V view"), (None, None, "K view")):
        _refused(_code(lib.kvhp_window_decode(P, k, v, P, P, 2, 8, 2, 64, 1000, 100, 4, P, 1 << 40,
                                              None)), kvhp.KVHP_ERR_INVALID, name)
        _refused(_code(lib.kvhp_window_prefill(P, k, v, P, P, P, P, 2, 10, 8, 2, 64, 1000, 100, 4,
                                               P, 1 << 40, None)), kvhp.KVHP_ERR_INVALID, name)
        _refused(_code(lib.kvhp_weighted_decode(P, k, v, P, None, P, P, P, 2, 8, 2, 64, 1000, 1, P,
                                                1 << 40, None)), kvhp.KVHP_ERR_INVALID, name)
    _refused(_code(lib.kvhp_prompt_weights(P, None, P, None, None, None, P, P, 2, 10, 8, 2, 64, 1000,
                                           0, 0, 1, P, 1 << 40, None)), kvhp.KVHP_ERR_INVALID,
             "K view")


def test_long_prompts_need_no_workspace():
    """A prompt of many rows fills the card by itself: its keys are not cut into ranges,
    however many they are."""
    lib = kvhp.load()
    for rows in (60000, 65536, 131072, 200000, 1 << 20):
        for d in (64, 128):
            assert lib.kvhp_window_prefill_workspace_bytes(1, rows, 32, 8, d, rows, 0, 0) == 0
