"""ctypes binding of libkvhp.so, the gfx950 KV-cache hot-path library.

The C ABI is declared in include/kvhp_c.h; this module mirrors it one to one
for Python callers (tests, bench, smoke).  Device memory and streams come from
torch: every tensor argument is a torch tensor on the GPU, every `stream` is a
torch.cuda.Stream (default: the current stream).  Errors raise KVHPError with
the library's kvhp_last_error() message, the Python counterpart of the
std::runtime_error the reference's CUDA_CHECK throws
(src/common/cuda_utils.h:12-21).

There is no CPU fallback: if the library is missing, load() raises.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libkvhp.so")
HEADER_PATH = os.path.join(os.path.dirname(_HERE), "include", "kvhp_c.h")

PAGE_SIZE = 16
KVHP_OK = 0
KVHP_ERR_INVALID = -1
KVHP_ERR_UNSUPPORTED = -2
KVHP_ERR_WORKSPACE = -3
KVHP_ERR_HIP = -4


class KVHPError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"kvhp error {code}: {msg}")
        self.code = code


class KVView(ctypes.Structure):
    """kvhp_kv_view: strided (block_table == NULL) or paged view of K or V."""

    _fields_ = [
        ("data", ctypes.c_void_p),
        ("stride_b", ctypes.c_int64),
        ("stride_h", ctypes.c_int64),
        ("stride_s", ctypes.c_int64),
        ("stride_d", ctypes.c_int64),
        ("block_table", ctypes.c_void_p),
        ("max_pages", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


_vp = ctypes.c_void_p
_i32 = ctypes.c_int
_i64 = ctypes.c_int64
_sz = ctypes.c_size_t
_f32 = ctypes.c_float
_u64 = ctypes.c_uint64

# name -> (restype, argtypes)
_SIGNATURES = {
    "kvhp_last_error": (ctypes.c_char_p, []),
    "kvhp_abi_version": (_i32, []),
    "kvhp_append_kv": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_paged_append_kv": (_i32, [_vp, _vp, _vp, _vp, _vp, _i32, _vp, _i32, _i32, _i32,
                                    _i32, _i32, _vp]),
    "kvhp_paged_gather_kv": (_i32, [_vp, _vp, _vp, _i32, _vp, _i32, _i32, _i32, _i32, _i32,
                                    _vp, _vp, _vp]),
    "kvhp_decode_auto_splits": (_i32, [_i32, _i32, _i32, _i32]),
    "kvhp_decode_workspace_bytes": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32]),
    "kvhp_decode_workspace_init": (_i32, [_vp, _sz, _vp]),
    "kvhp_decode_attention": (_i32, [_vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView), _vp,
                                     _vp, _i32, _i32, _i32, _i32, _i32, _i32, _vp, _sz, _vp]),
    "kvhp_build_id": (ctypes.c_char_p, []),
    "kvhp_stream_read": (_i32, [_vp, _sz, _vp, _vp]),
    "kvhp_page_read": (_i32, [_vp, _i64, _vp, _i64, _i32, _vp, _vp]),
    "kvhp_decode_attention_noalloc": (_i32, [_vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView),
                                             _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_paged_append_decode": (_i32, [_vp, _vp, _vp, ctypes.POINTER(KVView),
                                        ctypes.POINTER(KVView), _vp, _vp, _vp, _i32, _i32, _i32,
                                        _i32, _i32, _i32, _vp, _sz, _vp]),
    "kvhp_append_decode": (_i32, [_vp, _vp, _vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView),
                                  _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _vp, _sz,
                                  _vp]),
    "kvhp_decode_gqa": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_flash_prefill": (_i32, [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_flash_prefill_paged": (_i32, [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i32, _vp,
                                        _vp, _vp, _i32, _i32, _vp]),
    "kvhp_causal_gqa": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp]),
    # caches of bounded length
    "kvhp_window_decode_workspace_bytes": (_sz, [_i32] * 7),
    "kvhp_window_decode": (_i32, [_vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView), _vp, _vp,
                                  _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp, _sz, _vp]),
    "kvhp_window_prefill_workspace_bytes": (_sz, [_i32] * 8),
    "kvhp_window_prefill": (_i32, [_vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView), _vp, _vp,
                                   _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp,
                                   _sz, _vp]),
    "kvhp_weighted_decode_workspace_bytes": (_sz, [_i32] * 5),
    "kvhp_weighted_decode": (_i32, [_vp, ctypes.POINTER(KVView), ctypes.POINTER(KVView), _vp, _vp,
                                    _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _vp, _sz,
                                    _vp]),
    "kvhp_prompt_weights_workspace_bytes": (_sz, [_i32] * 6),
    "kvhp_prompt_weights": (_i32, [_vp, ctypes.POINTER(KVView), _vp, _vp, _vp, _vp, _vp, _vp,
                                   _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp,
                                   _sz, _vp]),
    "kvhp_evict_plan": (_i32, [_vp, _vp, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32,
                               _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_evict_apply": (_i32, [_vp, _vp, _vp, _vp, _vp, _i32, _vp, _vp, _i32, _i32, _i32, _i32,
                                _i32, _vp]),
    # appends that rotate, caches in 4 bits
    "kvhp_rope_append": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _f32, _vp, _vp,
                                _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_q4_page_bytes": (_sz, [_i32]),
    "kvhp_q4_rope_append": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _f32, _vp, _vp,
                                   _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_q4_gather": (_i32, [_vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32,
                              _vp]),
    "kvhp_q4_decode_workspace_bytes": (_sz, [_i32] * 5),
    "kvhp_q4_decode": (_i32, [_vp, _vp, _vp, _i32, _i32, _vp, _vp, _i32, _i32, _i32, _i32, _i32,
                              _vp, _sz, _vp]),
    "kvhp_q4_prefill_workspace_bytes": (_sz, [_i32] * 6),
    "kvhp_q4_prefill": (_i32, [_vp, _vp, _vp, _i32, _i32, _vp, _vp, _vp, _vp, _i32, _i32, _i32,
                               _i32, _i32, _i32, _vp, _sz, _vp]),
    # model operators
    "kvhp_gemv": (_i32, [_vp, _vp, _vp, _i32, _i32, _vp]),
    "kvhp_gemv_residual": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _vp]),
    "kvhp_rmsnorm_gemv": (_i32, [_vp, _vp, _vp, _f32, _vp, _vp, _i32, _i32, _vp]),
    "kvhp_rmsnorm_gemv_swiglu": (_i32, [_vp, _vp, _vp, _f32, _vp, _i32, _i32, _vp]),
    "kvhp_rmsnorm_qkv_rope_append": (_i32, [_vp, _vp, _vp, _f32, _vp, _f32, _vp, _vp, _vp, _vp,
                                            _i32, _i32, _i32, _i32, _i32, _i32, _vp]),
    "kvhp_gemv_residual_rows": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32, _vp]),
    "kvhp_gemv_rows_workspace_bytes": (_sz, [_i32, _i32, _i32]),
    "kvhp_gemv_residual_rows_ws": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32, _vp, _sz, _vp]),
    "kvhp_rmsnorm_gemv_rows": (_i32, [_vp, _vp, _vp, _f32, _vp, _vp, _i32, _i32, _i32, _vp]),
    "kvhp_rmsnorm_gemv_swiglu_rows": (_i32, [_vp, _vp, _vp, _f32, _vp, _i32, _i32, _i32, _vp]),
    "kvhp_rmsnorm_qkv_rope_append_rows": (_i32, [_vp, _vp, _vp, _f32, _vp, _f32, _vp, _vp, _vp,
                                                 _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
                                                 _vp]),
    "kvhp_rows_tiled_bytes": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32]),
    "kvhp_rows_tile_weights": (_i32, [_i32, _vp, _i32, _i32, _i32, _i32, _i32, _vp, _vp]),
    "kvhp_gemv_residual_rows_tiled": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32, _vp, _sz,
                                             _vp]),
    "kvhp_rmsnorm_gemv_rows_tiled": (_i32, [_vp, _vp, _vp, _f32, _vp, _vp, _i32, _i32, _i32,
                                            _vp]),
    "kvhp_rmsnorm_gemv_swiglu_rows_tiled": (_i32, [_vp, _vp, _vp, _f32, _vp, _i32, _i32, _i32,
                                                   _vp]),
    "kvhp_rmsnorm_qkv_rope_append_rows_tiled": (_i32, [_vp, _vp, _vp, _f32, _vp, _f32, _vp, _vp,
                                                       _vp, _vp, _i32, _i32, _i32, _i32, _i32,
                                                       _i32, _i32, _vp]),
    "kvhp_rmsnorm": (_i32, [_vp, _vp, _vp, _i64, _i64, _f32, _vp]),
    "kvhp_apply_rope": (_i32, [_vp, _vp, _i64, _i64, _i64, _i64, _i64, _f32, _vp]),
    "kvhp_split_qkv_rope": (_i32, [_vp, _i64, _i32, _i32, _i32, _i64, _f32, _vp, _vp, _vp, _vp]),
    "kvhp_split_qkv_rope_rows": (_i32, [_vp, _i64, _i32, _i32, _i32, _vp, _f32, _vp, _vp, _vp,
                                        _vp]),
    "kvhp_swiglu": (_i32, [_vp, _vp, _vp, _i64, _vp]),
    "kvhp_swiglu_rows": (_i32, [_vp, _vp, _i64, _i64, _vp]),
    "kvhp_embedding": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _vp]),
    "kvhp_argmax": (_i32, [_vp, _i64, _vp, _vp, _vp, _vp, _vp]),
    "kvhp_argmax_rows": (_i32, [_vp, _i64, _i64, _vp, _vp]),
    "kvhp_randn_f16": (_i32, [_vp, _i64, _u64, _u64, _f32, _vp]),
    "kvhp_fill_f16": (_i32, [_vp, _i64, _f32, _vp]),
    # model runner
    "kvhp_llama_create": (_i32, [_vp, _u64, _i32, ctypes.POINTER(ctypes.c_void_p)]),
    "kvhp_llama_destroy": (_i32, [_vp]),
    "kvhp_llama_prefill": (_i32, [_vp, _vp, _i32, _vp, _vp]),
    "kvhp_llama_decode_step": (_i32, [_vp, ctypes.c_int32, _vp, _vp]),
    "kvhp_llama_generate": (_i32, [_vp, _i32, _i32, _vp, _vp]),
    "kvhp_llama_tensor": (_i32, [_vp, _i32, _i32, ctypes.POINTER(ctypes.c_void_p),
                                 ctypes.POINTER(ctypes.c_size_t)]),
    "kvhp_llama_prefill_paged": (_i32, [_vp, _vp, _i32, _vp, _i32, _vp, _i32, _vp, _vp, _vp]),
    "kvhp_llama_prefill_cached": (_i32, [_vp, _vp, _i32, _i32, _vp, _i32, _vp, _vp, _i32, _vp,
                                         _vp, _vp]),
    "kvhp_llama_decode_paged": (_i32, [_vp, _vp, _i32, _vp, _i32, _vp, _i32, _vp, _vp, _i32,
                                       _vp, _vp, _vp]),
    "kvhp_llama_reserve": (_i32, [_vp, _i32, _i32]),
}

_lib: Optional[ctypes.CDLL] = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Load libkvhp.so (once).  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
    # torch's HIP runtime first, so that the library binds to the same one:
    # loaded the other way round, the process holds two HIP runtimes and the
    # library's finds no device once torch's has opened it.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(path)
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def exported_symbols() -> list:
    return list(_SIGNATURES)


def build_id() -> str:
    """Source hash the loaded library was linked with (kvhp_build_id)."""
    return load().kvhp_build_id().decode()


def source_build_id(root: str = os.path.dirname(os.path.abspath(__file__))) -> str:
    """The same hash over the sources in this tree (Makefile ID_SRCS): the
    library matches the tree when build_id() == source_build_id()."""
    import glob
    import hashlib
    csrc = os.path.join(root, "csrc")
    files = (sorted(glob.glob(os.path.join(csrc, "*.hip"))) +
             sorted(glob.glob(os.path.join(csrc, "*.h"))) +
             [os.path.join(root, "..", "include", "kvhp_c.h")])
    h = hashlib.sha256()
    for f in files:
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


def stream_read(buf, sink, stream=None):
    """Streaming read of the whole tensor `buf` (kvhp_stream_read); sink: a
    device tensor of at least 4 bytes."""
    _check(load().kvhp_stream_read(_ptr(buf), buf.numel() * buf.element_size(), _ptr(sink),
                                   _stream(stream)))


def page_read(pool, page_ids, page_bytes, sink, stream=None):
    """Read the pages page_ids (int32 device tensor) of the device tensor
    `pool` cut into pages of page_bytes (kvhp_page_read); sink: a 4-byte
    device tensor."""
    _check(load().kvhp_page_read(_ptr(pool), pool.numel() * pool.element_size(), _ptr(page_ids),
                                 page_ids.numel(), page_bytes, _ptr(sink), _stream(stream)))


def last_error() -> str:
    return load().kvhp_last_error().decode()


def _check(rc: int) -> None:
    if rc != KVHP_OK:
        raise KVHPError(rc, last_error())


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    return t.data_ptr()


_raw_stream = None    # torch's (device index) -> current stream's handle, once a call was made
_raw_device = None    # and its current device's index


def _first_stream() -> int:
    """torch's current stream, through torch's own initialisation of the device
    (and its refusal of forked children); later calls take the handle without
    building a torch.cuda.Stream object around it (0.2 against 2.8 us, a third of
    a small call's host time)."""
    global _raw_stream, _raw_device
    import torch   # here: importing this module loads no torch
    handle = torch.cuda.current_stream().cuda_stream
    _raw_device = getattr(torch._C, "_cuda_getDevice", None)   # not public names
    if _raw_device is not None:
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return handle


def _forget_stream() -> None:
    global _raw_stream
    _raw_stream = None


os.register_at_fork(after_in_child=_forget_stream)


def _stream(stream) -> Optional[int]:
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        return _first_stream()
    return _raw_stream(_raw_device())


# ----------------------------------------------------------------- views --
def strided_view(t, stride_b: int, stride_h: int, stride_s: int, stride_d: int = 1) -> KVView:
    v = KVView()
    v.data = t.data_ptr()
    v.stride_b, v.stride_h, v.stride_s, v.stride_d = stride_b, stride_h, stride_s, stride_d
    v.block_table = None
    v.max_pages = v.page_size = v.num_pages = 0
    return v


def paged_view(pool, block_tables) -> KVView:
    """View over a pool [Hkv][P][16][D] with int32 block tables [B][max_pages]."""
    hkv, p, page, d = pool.shape
    assert page == PAGE_SIZE
    v = KVView()
    v.data = pool.data_ptr()
    v.stride_b = 0
    v.stride_h = p * page * d
    v.stride_s = d
    v.stride_d = 1
    v.block_table = block_tables.data_ptr()
    v.max_pages = block_tables.shape[1]
    v.page_size = page
    v.num_pages = p
    return v


# ------------------------------------------------------------- entry pts --
def append_kv(src_k, src_v, dst_k, dst_v, num_tokens, start_pos, num_kv_heads, max_seq,
              head_dim, stream=None):
    _check(load().kvhp_append_kv(_ptr(src_k), _ptr(src_v), _ptr(dst_k), _ptr(dst_v),
                                 num_tokens, start_pos, num_kv_heads, max_seq, head_dim,
                                 _stream(stream)))


def paged_append_kv(src_k, src_v, pool_k, pool_v, block_tables, start_pos, batch, num_tokens,
                    num_kv_heads, head_dim, stream=None):
    _check(load().kvhp_paged_append_kv(
        _ptr(src_k), _ptr(src_v), _ptr(pool_k), _ptr(pool_v), _ptr(block_tables),
        block_tables.shape[1], _ptr(start_pos), batch, num_tokens, num_kv_heads, head_dim,
        pool_k.shape[1], _stream(stream)))


def paged_gather_kv(pool_k, pool_v, block_tables, seq_lens, max_len, out_k, out_v,
                    stream=None):
    hkv, p, _, d = pool_k.shape
    _check(load().kvhp_paged_gather_kv(
        _ptr(pool_k), _ptr(pool_v), _ptr(block_tables), block_tables.shape[1], _ptr(seq_lens),
        seq_lens.shape[0], hkv, d, p, max_len, _ptr(out_k), _ptr(out_v), _stream(stream)))


def decode_auto_splits(batch, num_kv_heads, head_dim, max_seq_len) -> int:
    return load().kvhp_decode_auto_splits(batch, num_kv_heads, head_dim, max_seq_len)


def decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                           num_splits=0) -> int:
    return load().kvhp_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim,
                                              max_seq_len, num_splits)


def decode_workspace_init(ws, stream=None):
    _check(load().kvhp_decode_workspace_init(_ptr(ws), ws.numel() * ws.element_size(),
                                             _stream(stream)))


def decode_attention(q, k_view: KVView, v_view: KVView, seq_lens, out, num_q_heads,
                     num_kv_heads, head_dim, max_seq_len, num_splits=0, workspace=None,
                     stream=None):
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(load().kvhp_decode_attention(
        _ptr(q), ctypes.byref(k_view), ctypes.byref(v_view), _ptr(seq_lens), _ptr(out),
        seq_lens.shape[0], num_q_heads, num_kv_heads, head_dim, max_seq_len, num_splits,
        _ptr(workspace), ws_bytes, _stream(stream)))


def decode_attention_noalloc(q, k_view: KVView, v_view: KVView, seq_lens, out, num_q_heads,
                             num_kv_heads, head_dim, max_seq_len, num_splits=0, stream=None):
    """decode_attention with the split partials in the library's static
    device scratch (no allocation; calls overlapping on one GPU race)."""
    _check(load().kvhp_decode_attention_noalloc(
        _ptr(q), ctypes.byref(k_view), ctypes.byref(v_view), _ptr(seq_lens), _ptr(out),
        seq_lens.shape[0], num_q_heads, num_kv_heads, head_dim, max_seq_len, num_splits,
        _stream(stream)))


def paged_append_decode(q, k_new, v_new, k_view: KVView, v_view: KVView, positions, seq_lens,
                        out, num_q_heads, num_kv_heads, head_dim, max_seq_len, num_splits=0,
                        workspace=None, stream=None):
    """Append row b of k_new / v_new [B][Hkv][D] at positions[b], then decode
    attention over seq_lens[b] keys (one call; paged views)."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(load().kvhp_paged_append_decode(
        _ptr(q), _ptr(k_new), _ptr(v_new), ctypes.byref(k_view), ctypes.byref(v_view),
        _ptr(positions), _ptr(seq_lens), _ptr(out), seq_lens.shape[0], num_q_heads,
        num_kv_heads, head_dim, max_seq_len, num_splits, _ptr(workspace), ws_bytes,
        _stream(stream)))


def append_decode(q, k_new, v_new, k_view: KVView, v_view: KVView, positions, seq_lens, out,
                  num_q_heads, num_kv_heads, head_dim, max_seq_len, num_splits=0, workspace=None,
                  stream=None):
    """paged_append_decode for views of either kind (strided views: row
    positions[b] of sequence b, dropped outside [0, max_seq_len))."""
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(load().kvhp_append_decode(
        _ptr(q), _ptr(k_new), _ptr(v_new), ctypes.byref(k_view), ctypes.byref(v_view),
        _ptr(positions), _ptr(seq_lens), _ptr(out), seq_lens.shape[0], num_q_heads,
        num_kv_heads, head_dim, max_seq_len, num_splits, _ptr(workspace), ws_bytes,
        _stream(stream)))


def decode_gqa(q, k_cache, v_cache, out, total_seq_len, num_q_heads, num_kv_heads, max_seq,
               head_dim, stream=None):
    _check(load().kvhp_decode_gqa(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                  total_seq_len, num_q_heads, num_kv_heads, max_seq, head_dim,
                                  _stream(stream)))


def flash_prefill(q, k, v, out, seq_len, num_q_heads, num_kv_heads, head_dim, batch=1,
                  stream=None):
    _check(load().kvhp_flash_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(out), seq_len,
                                     num_q_heads, num_kv_heads, head_dim, batch,
                                     _stream(stream)))


def flash_prefill_paged(q, k, v, out, seq_len, num_q_heads, num_kv_heads, head_dim, batch,
                        pool_k, pool_v, block_tables, stream=None):
    _check(load().kvhp_flash_prefill_paged(
        _ptr(q), _ptr(k), _ptr(v), _ptr(out), seq_len, num_q_heads, num_kv_heads, head_dim,
        batch, _ptr(pool_k), _ptr(pool_v), _ptr(block_tables), block_tables.shape[1],
        pool_k.shape[1], _stream(stream)))


def causal_gqa(q, k, v, out, seq_len, num_q_heads, num_kv_heads, head_dim, stream=None):
    _check(load().kvhp_causal_gqa(_ptr(q), _ptr(k), _ptr(v), _ptr(out), seq_len, num_q_heads,
                                  num_kv_heads, head_dim, _stream(stream)))


# --------------------------------------------- caches of bounded length --
def _bytes(ws) -> int:
    return 0 if ws is None else ws.nbytes


def window_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                                  window, sinks=0) -> int:
    return load().kvhp_window_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim,
                                                     max_seq_len, window, sinks)


def window_decode(q, k_view: KVView, v_view: KVView, seq_lens, out, num_q_heads, num_kv_heads,
                  head_dim, max_seq_len, window, sinks=0, workspace=None, stream=None):
    """decode_attention over each sequence's last `window` keys and its first
    `sinks` ones (window 0: every key); workspace: a tensor of
    window_decode_workspace_bytes bytes."""
    _check(load().kvhp_window_decode(
        _ptr(q), ctypes.byref(k_view), ctypes.byref(v_view), _ptr(seq_lens), _ptr(out),
        seq_lens.shape[0], num_q_heads, num_kv_heads, head_dim, max_seq_len, window, sinks,
        _ptr(workspace), _bytes(workspace), _stream(stream)))


def window_prefill_workspace_bytes(batch, rows, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                                   window, sinks=0) -> int:
    return load().kvhp_window_prefill_workspace_bytes(batch, rows, num_q_heads, num_kv_heads,
                                                      head_dim, max_seq_len, window, sinks)


def window_prefill(q, k_view: KVView, v_view: KVView, out, num_q_heads, num_kv_heads, head_dim,
                   max_seq_len, window, sinks=0, q_start=None, seq_lens=None, lse=None,
                   workspace=None, stream=None):
    """Rows q [B][rows][Hq][D] at positions q_start[b] + r over the views' first
    seq_lens[b] keys; out as q, lse fp32 [B][Hq][rows] (optional); padding rows
    are left as they were."""
    _check(load().kvhp_window_prefill(
        _ptr(q), ctypes.byref(k_view), ctypes.byref(v_view), _ptr(q_start), _ptr(seq_lens),
        _ptr(out), _ptr(lse), q.shape[0], q.shape[1], num_q_heads, num_kv_heads, head_dim,
        max_seq_len, window, sinks, _ptr(workspace), _bytes(workspace), _stream(stream)))


def weighted_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim,
                                    max_seq_len) -> int:
    return load().kvhp_weighted_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim,
                                                       max_seq_len)


def weighted_decode(q, k_view: KVView, v_view: KVView, seq_lens, out, weights, num_q_heads,
                    num_kv_heads, head_dim, max_seq_len, new_keys=1, ages=None, newest=None,
                    workspace=None, stream=None):
    """decode_attention that adds every key's attention weight, summed over its
    KV head's query heads, to its slot of weights (fp32 [Hkv][P][16]); the last
    new_keys keys start from zero and get their age (int32 [Hkv][P][16])."""
    _check(load().kvhp_weighted_decode(
        _ptr(q), ctypes.byref(k_view), ctypes.byref(v_view), _ptr(seq_lens), _ptr(newest),
        _ptr(out), _ptr(weights), _ptr(ages), seq_lens.shape[0], num_q_heads, num_kv_heads,
        head_dim, max_seq_len, new_keys, _ptr(workspace), _bytes(workspace), _stream(stream)))


def prompt_weights_workspace_bytes(batch, rows, num_q_heads, num_kv_heads, head_dim,
                                   max_seq_len) -> int:
    return load().kvhp_prompt_weights_workspace_bytes(batch, rows, num_q_heads, num_kv_heads,
                                                      head_dim, max_seq_len)


def prompt_weights(q, k_view: KVView, lse, weights, num_q_heads, num_kv_heads, head_dim,
                   max_seq_len, new_keys, window=0, sinks=0, q_start=None, seq_lens=None,
                   ages=None, newest=None, workspace=None, stream=None):
    """Adds to weights the attention that the rows q [B][rows][Hq][D] give each
    key, from the lse that window_prefill left for them."""
    _check(load().kvhp_prompt_weights(
        _ptr(q), ctypes.byref(k_view), _ptr(lse), _ptr(q_start), _ptr(seq_lens), _ptr(newest),
        _ptr(weights), _ptr(ages), q.shape[0], q.shape[1], num_q_heads, num_kv_heads, head_dim,
        max_seq_len, window, sinks, new_keys, _ptr(workspace), _bytes(workspace),
        _stream(stream)))


def evict_plan(weights, ages, block_tables, seq_lens, moves, counts, new_lens, max_seq_len,
               budget, sinks=0, recent=0, newest=None, stream=None):
    """The moves [B][Hkv][max_moves][2], counts [B][Hkv] and new_lens [B] that cut
    each sequence to its budget of slots (weights, ages: [Hkv][P][16])."""
    _check(load().kvhp_evict_plan(
        _ptr(weights), _ptr(ages), _ptr(block_tables), block_tables.shape[1], _ptr(seq_lens),
        _ptr(newest), _ptr(moves), _ptr(counts), _ptr(new_lens), seq_lens.shape[0],
        weights.shape[0], weights.shape[1], max_seq_len, budget, sinks, recent, moves.shape[2],
        _stream(stream)))


def evict_apply(pool_k, pool_v, weights, ages, block_tables, moves, counts, stream=None):
    """Carries out evict_plan's moves on pools [Hkv][P][16][D] and on the sums."""
    hkv, pages, _, d = pool_k.shape
    _check(load().kvhp_evict_apply(
        _ptr(pool_k), _ptr(pool_v), _ptr(weights), _ptr(ages), _ptr(block_tables),
        block_tables.shape[1], _ptr(moves), _ptr(counts), counts.shape[0], hkv, d, pages,
        moves.shape[2], _stream(stream)))


# ------------------------- appends that rotate, caches held in 4 bits --
def _token_rows(t, what):
    """(batch, rows, stride) of q, k or v [B][rows][H][D]: consecutive tokens stride
    halfs apart, the heads of a token in a row."""
    B, R, H, D = t.shape
    sb, sr, sh, sd = t.stride()
    step = sr if R > 1 else sb if B > 1 else H * D   # a dimension of one has no stride
    if (D > 1 and sd != 1) or (H > 1 and sh != D) or (R > 1 and B > 1 and sb != R * sr):
        raise KVHPError(KVHP_ERR_INVALID,
                        f"{what}: tokens of rows [H][D] at one stride wanted, got strides "
                        f"{tuple(t.stride())} of shape {tuple(t.shape)}")
    return B, R, step


def _append_rows(q, k, v, q_out, what, heads=None):
    """(batch, rows, q_stride, k_stride, v_stride) of an append's tensors, of `heads` =
    (num_q_heads, num_kv_heads, head_dim)."""
    shape = k.shape
    B, R, H, D = shape
    same = v.shape == shape and (heads is None or H == heads[1] and D == heads[2])
    kb, sk, kh, kd = k.stride()
    vb, sv, vh, vd = v.stride()
    # as slices of contiguous tensors are; others by _token_rows, which knows what it can take
    if not (kd == vd == 1 and kh == vh == D and kb == R * sk and vb == R * sv):
        sk, sv = _token_rows(k, what)[2], _token_rows(v, what)[2]
    sq = 0
    if q is not None:
        qb, sq, qh, qd = q.stride()
        if not (qd == 1 and qh == D and qb == R * sq):
            sq = _token_rows(q, what)[2]
        qs = q.shape
        same = (same and qs[0] == B and qs[1] == R and qs[3] == D
                and (heads is None or qs[2] == heads[0]))
        if q_out is not None:
            same = same and q_out.shape == qs
    if not same:
        raise KVHPError(KVHP_ERR_INVALID, f"{what}: q, k, v and q_out of different rows"
                                          + (f", or of others than {heads} heads and dims" if heads else ""))
    if q_out is not None and not q_out.is_contiguous():
        raise KVHPError(KVHP_ERR_INVALID, f"{what}: q_out must be contiguous")
    return B, R, sq, sk, sv


def _refuse_sizes(what, whole, sequences, n):
    """The library takes addresses and goes by the numbers it is called with.  Raises for the
    first of `whole`, name: (tensor or None, values), that is not contiguous or holds another
    number of values (block tables: fewer), or of `sequences` that has no value for each of
    n.  Called where a call's own check of all of them failed."""
    for name, (t, values) in whole.items():
        if t is None:
            continue
        got = t.numel()
        if got < values or (got > values and name != "block_tables") or not t.is_contiguous():
            raise KVHPError(KVHP_ERR_INVALID, f"{what}: {name}: {values} contiguous values wanted, got "
                                              f"{tuple(t.shape)} with strides {t.stride()}")
    for name, t in sequences.items():
        if t is not None and (t.numel() < n or not t.is_contiguous()):
            raise KVHPError(KVHP_ERR_INVALID, f"{what}: {name}: a value for each of {n} sequences wanted, got "
                                              f"{tuple(t.shape)} with strides {t.stride()}")


def rope_append(q, k, v, positions, q_out, pool_k, pool_v, block_tables, num_q_heads,
                num_kv_heads, head_dim, theta, slots=None, seq_lens=None, stream=None):
    """Rotates rows q [B][rows][Hq][D] (to q_out) and k [B][rows][Hkv][D] to text
    positions positions[b] + r and writes K and V to slots slots[b] + r of the pools
    [Hkv][P][16][D].  q, k, v may be parts of one fused projection; theta 0: no rotation."""
    B, R, sq, sk, sv = _append_rows(q, k, v, q_out, "rope_append", (num_q_heads, num_kv_heads, head_dim))
    max_pages, pages = block_tables.shape[1], pool_k.shape[1]
    pooled = num_kv_heads * pages * PAGE_SIZE * head_dim
    if not (pool_k.numel() == pooled == pool_v.numel() and block_tables.numel() >= B * max_pages
            and (positions is None or positions.numel() >= B and positions.is_contiguous())
            and (slots is None or slots.numel() >= B and slots.is_contiguous())
            and (seq_lens is None or seq_lens.numel() >= B and seq_lens.is_contiguous())
            and pool_k.is_contiguous() and pool_v.is_contiguous() and block_tables.is_contiguous()):
        _refuse_sizes("rope_append", {"pool_k": (pool_k, pooled), "pool_v": (pool_v, pooled),
                                      "block_tables": (block_tables, B * max_pages)},
                      {"positions": positions, "slots": slots, "seq_lens": seq_lens}, B)
    _check(load().kvhp_rope_append(
        _ptr(q), k.data_ptr(), v.data_ptr(), sq, sk, sv, _ptr(positions), _ptr(slots), _ptr(seq_lens),
        theta, _ptr(q_out), pool_k.data_ptr(), pool_v.data_ptr(), block_tables.data_ptr(),
        max_pages, pages, B, R, num_q_heads, num_kv_heads, head_dim, _stream(stream)))


def q4_page_bytes(head_dim) -> int:
    """Bytes of a 4-bit page (16 tokens' K and V of one KV head)."""
    return load().kvhp_q4_page_bytes(head_dim)


def q4_rope_append(q, k, v, positions, q_out, pool, block_tables, num_q_heads, num_kv_heads,
                   head_dim, theta, slots=None, seq_lens=None, stream=None):
    """rope_append into a 4-bit pool, uint8 [Hkv][P][q4_page_bytes(D)]."""
    B, R, sq, sk, sv = _append_rows(q, k, v, q_out, "q4_rope_append", (num_q_heads, num_kv_heads, head_dim))
    max_pages, pages = block_tables.shape[1], pool.shape[1]
    pooled = num_kv_heads * pages * PAGE_SIZE * (head_dim + 8)
    if not (pool.numel() == pooled and block_tables.numel() >= B * max_pages
            and (positions is None or positions.numel() >= B and positions.is_contiguous())
            and (slots is None or slots.numel() >= B and slots.is_contiguous())
            and (seq_lens is None or seq_lens.numel() >= B and seq_lens.is_contiguous())
            and pool.is_contiguous() and block_tables.is_contiguous()):
        _refuse_sizes("q4_rope_append", {"pool": (pool, pooled), "block_tables": (block_tables, B * max_pages)},
                      {"positions": positions, "slots": slots, "seq_lens": seq_lens}, B)
    _check(load().kvhp_q4_rope_append(
        _ptr(q), k.data_ptr(), v.data_ptr(), sq, sk, sv, _ptr(positions), _ptr(slots), _ptr(seq_lens),
        theta, _ptr(q_out), pool.data_ptr(), block_tables.data_ptr(), max_pages, pages,
        B, R, num_q_heads, num_kv_heads, head_dim, _stream(stream)))


def q4_gather(pool, block_tables, seq_lens, out_k, out_v, start=None, stream=None):
    """Positions start[b] + t of a 4-bit pool as fp16 [B][Hkv][max_len][D] (either output
    may be None), zeros from seq_lens[b] on."""
    B, hkv, n, d = (out_k if out_k is not None else out_v).shape
    max_pages, pages = block_tables.shape[1], pool.shape[1]
    values, pooled = B * hkv * n * d, hkv * pages * PAGE_SIZE * (d + 8)
    if not (pool.numel() == pooled and block_tables.numel() >= B * max_pages
            and (out_k is None or out_k.is_contiguous())
            and (out_v is None or out_v.numel() == values and out_v.is_contiguous())
            and seq_lens.numel() >= B and seq_lens.is_contiguous()
            and (start is None or start.numel() >= B and start.is_contiguous())
            and pool.is_contiguous() and block_tables.is_contiguous()):
        _refuse_sizes("q4_gather", {"out_k": (out_k, values), "out_v": (out_v, values), "pool": (pool, pooled),
                                    "block_tables": (block_tables, B * max_pages)},
                      {"seq_lens": seq_lens, "start": start}, B)
    _check(load().kvhp_q4_gather(
        pool.data_ptr(), block_tables.data_ptr(), max_pages, pages, _ptr(start),
        seq_lens.data_ptr(), _ptr(out_k), _ptr(out_v), B, hkv, d, n, _stream(stream)))


def q4_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len) -> int:
    return load().kvhp_q4_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim,
                                                 max_seq_len)


def q4_decode(q, pool, block_tables, seq_lens, out, num_q_heads, num_kv_heads, head_dim,
              max_seq_len, workspace=None, stream=None):
    """decode_attention over a 4-bit pool; workspace: a tensor of
    q4_decode_workspace_bytes bytes."""
    B, max_pages, pages = seq_lens.shape[0], block_tables.shape[1], pool.shape[1]
    values, pooled = B * num_q_heads * head_dim, num_kv_heads * pages * PAGE_SIZE * (head_dim + 8)
    if not (q.numel() == values == out.numel() and pool.numel() == pooled
            and block_tables.numel() >= B * max_pages
            and q.is_contiguous() and out.is_contiguous() and seq_lens.is_contiguous()
            and pool.is_contiguous() and block_tables.is_contiguous()):
        _refuse_sizes("q4_decode", {"q": (q, values), "out": (out, values), "pool": (pool, pooled),
                                    "block_tables": (block_tables, B * max_pages)}, {"seq_lens": seq_lens}, B)
    _check(load().kvhp_q4_decode(
        q.data_ptr(), pool.data_ptr(), block_tables.data_ptr(), max_pages, pages,
        seq_lens.data_ptr(), out.data_ptr(), B, num_q_heads, num_kv_heads, head_dim,
        max_seq_len, _ptr(workspace), _bytes(workspace), _stream(stream)))


def q4_prefill_workspace_bytes(batch, rows, num_q_heads, num_kv_heads, head_dim,
                               max_seq_len) -> int:
    return load().kvhp_q4_prefill_workspace_bytes(batch, rows, num_q_heads, num_kv_heads,
                                                  head_dim, max_seq_len)


def q4_prefill(q, pool, block_tables, out, num_q_heads, num_kv_heads, head_dim, max_seq_len,
               q_start=None, seq_lens=None, lse=None, workspace=None, stream=None):
    """Rows q [B][rows][Hq][D] at positions q_start[b] + r, each over the keys of the 4-bit
    pool up to itself; out as q, lse fp32 [B][Hq][rows] (optional); padding rows are left
    as they were."""
    B, R, _, _ = q.shape
    max_pages, pages = block_tables.shape[1], pool.shape[1]
    values, pooled = B * R * num_q_heads * head_dim, num_kv_heads * pages * PAGE_SIZE * (head_dim + 8)
    if not (q.numel() == values == out.numel() and pool.numel() == pooled
            and block_tables.numel() >= B * max_pages
            and (lse is None or lse.numel() == B * R * num_q_heads and lse.is_contiguous())
            and (q_start is None or q_start.numel() >= B and q_start.is_contiguous())
            and (seq_lens is None or seq_lens.numel() >= B and seq_lens.is_contiguous())
            and q.is_contiguous() and out.is_contiguous() and pool.is_contiguous()
            and block_tables.is_contiguous()):
        _refuse_sizes("q4_prefill", {"q": (q, values), "out": (out, values), "pool": (pool, pooled),
                                     "lse": (lse, B * R * num_q_heads),
                                     "block_tables": (block_tables, B * max_pages)},
                      {"q_start": q_start, "seq_lens": seq_lens}, B)
    _check(load().kvhp_q4_prefill(
        q.data_ptr(), pool.data_ptr(), block_tables.data_ptr(), max_pages, pages,
        _ptr(q_start), _ptr(seq_lens), out.data_ptr(), _ptr(lse), B, R, num_q_heads,
        num_kv_heads, head_dim, max_seq_len, _ptr(workspace), _bytes(workspace),
        _stream(stream)))


# ------------------------------------------------------ model operators --
def gemv(W, x, y, N, K, stream=None):
    _check(load().kvhp_gemv(_ptr(W), _ptr(x), _ptr(y), N, K, _stream(stream)))


def gemv_residual(W, x, r, y, N, K, stream=None):
    _check(load().kvhp_gemv_residual(_ptr(W), _ptr(x), _ptr(r), _ptr(y), N, K, _stream(stream)))


def rmsnorm_gemv(W, x, norm_w, eps, N, K, y16=None, y32=None, stream=None):
    _check(load().kvhp_rmsnorm_gemv(_ptr(W), _ptr(x), _ptr(norm_w), eps, _ptr(y16), _ptr(y32), N,
                                    K, _stream(stream)))


def rmsnorm_gemv_swiglu(W_gate_up, x, norm_w, eps, out, N, K, stream=None):
    _check(load().kvhp_rmsnorm_gemv_swiglu(_ptr(W_gate_up), _ptr(x), _ptr(norm_w), eps, _ptr(out),
                                           N, K, _stream(stream)))


def rmsnorm_qkv_rope_append(W_qkv, x, norm_w, eps, seq_len, theta, q_out, pool_k, pool_v,
                            block_table, num_q_heads, num_kv_heads, head_dim, K, stream=None):
    """pool_k / pool_v [Hkv][P][16][D]; block_table int32 [max_pages] (one sequence)."""
    _check(load().kvhp_rmsnorm_qkv_rope_append(
        _ptr(W_qkv), _ptr(x), _ptr(norm_w), eps, _ptr(seq_len), theta, _ptr(q_out), _ptr(pool_k),
        _ptr(pool_v), _ptr(block_table), block_table.numel(), pool_k.shape[1], num_q_heads,
        num_kv_heads, head_dim, K, _stream(stream)))


def gemv_residual_rows(W, x, r, y, N, K, batch, stream=None):
    _check(load().kvhp_gemv_residual_rows(_ptr(W), _ptr(x), _ptr(r), _ptr(y), N, K, batch,
                                          _stream(stream)))


def gemv_rows_workspace_bytes(N, K, batch):
    return load().kvhp_gemv_rows_workspace_bytes(N, K, batch)


def gemv_residual_rows_ws(W, x, r, y, N, K, batch, workspace=None, stream=None):
    """gemv_residual_rows with a caller workspace (uint8 tensor): large
    batches split over K; bit-identical output."""
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _check(load().kvhp_gemv_residual_rows_ws(_ptr(W), _ptr(x), _ptr(r), _ptr(y), N, K, batch,
                                             _ptr(workspace), nbytes, _stream(stream)))


def rmsnorm_gemv_rows(W, x, norm_w, eps, N, K, batch, y16=None, y32=None, stream=None):
    _check(load().kvhp_rmsnorm_gemv_rows(_ptr(W), _ptr(x), _ptr(norm_w), eps, _ptr(y16),
                                         _ptr(y32), N, K, batch, _stream(stream)))


def rmsnorm_gemv_swiglu_rows(W_gate_up, x, norm_w, eps, out, N, K, batch, stream=None):
    _check(load().kvhp_rmsnorm_gemv_swiglu_rows(_ptr(W_gate_up), _ptr(x), _ptr(norm_w), eps,
                                                _ptr(out), N, K, batch, _stream(stream)))


def rmsnorm_qkv_rope_append_rows(W_qkv, x, norm_w, eps, positions, theta, q_out, pool_k, pool_v,
                                 block_tables, num_q_heads, num_kv_heads, head_dim, K, batch,
                                 stream=None):
    """pool_k / pool_v [Hkv][P][16][D]; block_tables int32 [batch][max_pages]."""
    _check(load().kvhp_rmsnorm_qkv_rope_append_rows(
        _ptr(W_qkv), _ptr(x), _ptr(norm_w), eps, _ptr(positions), theta, _ptr(q_out),
        _ptr(pool_k), _ptr(pool_v), _ptr(block_tables), block_tables.shape[1], pool_k.shape[1],
        num_q_heads, num_kv_heads, head_dim, K, batch, _stream(stream)))


ROWS_PLAIN, ROWS_SWIGLU, ROWS_QKV = 0, 1, 2


def rows_tiled_bytes(kind, N, K, num_q_heads=0, num_kv_heads=0, head_dim=0):
    return load().kvhp_rows_tiled_bytes(kind, N, K, num_q_heads, num_kv_heads, head_dim)


def rows_tile_weights(kind, W, N, K, W_tiled, num_q_heads=0, num_kv_heads=0, head_dim=0,
                      stream=None):
    """Copy row-major W into the batched projections' tiled layout (W_tiled:
    rows_tiled_bytes bytes, any dtype)."""
    _check(load().kvhp_rows_tile_weights(kind, _ptr(W), N, K, num_q_heads, num_kv_heads,
                                         head_dim, _ptr(W_tiled), _stream(stream)))


def gemv_residual_rows_tiled(Wt, x, r, y, N, K, batch, workspace=None, stream=None):
    nbytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _check(load().kvhp_gemv_residual_rows_tiled(_ptr(Wt), _ptr(x), _ptr(r), _ptr(y), N, K, batch,
                                                _ptr(workspace), nbytes, _stream(stream)))


def rmsnorm_gemv_rows_tiled(Wt, x, norm_w, eps, N, K, batch, y16=None, y32=None, stream=None):
    _check(load().kvhp_rmsnorm_gemv_rows_tiled(_ptr(Wt), _ptr(x), _ptr(norm_w), eps, _ptr(y16),
                                               _ptr(y32), N, K, batch, _stream(stream)))


def rmsnorm_gemv_swiglu_rows_tiled(Wt, x, norm_w, eps, out, N, K, batch, stream=None):
    _check(load().kvhp_rmsnorm_gemv_swiglu_rows_tiled(_ptr(Wt), _ptr(x), _ptr(norm_w), eps,
                                                      _ptr(out), N, K, batch, _stream(stream)))


def rmsnorm_qkv_rope_append_rows_tiled(Wt, x, norm_w, eps, positions, theta, q_out, pool_k,
                                       pool_v, block_tables, num_q_heads, num_kv_heads, head_dim,
                                       K, batch, stream=None):
    _check(load().kvhp_rmsnorm_qkv_rope_append_rows_tiled(
        _ptr(Wt), _ptr(x), _ptr(norm_w), eps, _ptr(positions), theta, _ptr(q_out),
        _ptr(pool_k), _ptr(pool_v), _ptr(block_tables), block_tables.shape[1], pool_k.shape[1],
        num_q_heads, num_kv_heads, head_dim, K, batch, _stream(stream)))


def rmsnorm(x, weight, out, rows, dim, eps, stream=None):
    _check(load().kvhp_rmsnorm(_ptr(x), _ptr(weight), _ptr(out), rows, dim, eps, _stream(stream)))


def apply_rope(q, k, seq_len, num_q_heads, num_kv_heads, head_dim, start_pos, theta, stream=None):
    _check(load().kvhp_apply_rope(_ptr(q), _ptr(k), seq_len, num_q_heads, num_kv_heads, head_dim,
                                  start_pos, theta, _stream(stream)))


def split_qkv_rope(qkv, seq_len, num_q_heads, num_kv_heads, head_dim, start_pos, theta, q, k, v,
                   stream=None):
    _check(load().kvhp_split_qkv_rope(_ptr(qkv), seq_len, num_q_heads, num_kv_heads, head_dim,
                                      start_pos, theta, _ptr(q), _ptr(k), _ptr(v),
                                      _stream(stream)))


def split_qkv_rope_rows(qkv, rows, num_q_heads, num_kv_heads, head_dim, positions, theta, q, k,
                        v, stream=None):
    _check(load().kvhp_split_qkv_rope_rows(_ptr(qkv), rows, num_q_heads, num_kv_heads, head_dim,
                                           _ptr(positions), theta, _ptr(q), _ptr(k), _ptr(v),
                                           _stream(stream)))


def swiglu(gate, up, out, count, stream=None):
    _check(load().kvhp_swiglu(_ptr(gate), _ptr(up), _ptr(out), count, _stream(stream)))


def swiglu_rows(gate_up, out, rows, n, stream=None):
    _check(load().kvhp_swiglu_rows(_ptr(gate_up), _ptr(out), rows, n, _stream(stream)))


def embedding(token_ids, table, out, n, hidden, vocab, stream=None):
    _check(load().kvhp_embedding(_ptr(token_ids), _ptr(table), _ptr(out), n, hidden, vocab,
                                 _stream(stream)))


def argmax(logits, n, token, seq_len=None, log=None, log_count=None, stream=None):
    _check(load().kvhp_argmax(_ptr(logits), n, _ptr(token), _ptr(seq_len), _ptr(log),
                              _ptr(log_count), _stream(stream)))


def argmax_rows(logits, rows, n, tokens, stream=None):
    _check(load().kvhp_argmax_rows(_ptr(logits), rows, n, _ptr(tokens), _stream(stream)))


def randn_f16(out, seed, stream_id, std, stream=None):
    _check(load().kvhp_randn_f16(_ptr(out), out.numel(), seed, stream_id, std, _stream(stream)))


def fill_f16(out, value, stream=None):
    _check(load().kvhp_fill_f16(_ptr(out), out.numel(), value, _stream(stream)))


# ------------------------------------------------------------ model runner --
class LlamaConfig(ctypes.Structure):
    """kvhp_llama_config."""

    _fields_ = [("vocab_size", ctypes.c_int), ("hidden_size", ctypes.c_int),
                ("num_layers", ctypes.c_int), ("num_q_heads", ctypes.c_int),
                ("num_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("ffn_size", ctypes.c_int), ("rms_eps", ctypes.c_float),
                ("rope_theta", ctypes.c_float), ("reserved", ctypes.c_int)]


def llama_1b_config() -> LlamaConfig:
    """22 layers, hidden 2048, 32 q / 4 KV heads of 64,
    SwiGLU 5632, vocab 32000, RMSNorm eps 1e-5, RoPE theta 10000."""
    return LlamaConfig(32000, 2048, 22, 32, 4, 64, 5632, 1e-5, 10000.0, 0)


LLAMA_EMBED, LLAMA_LM_HEAD, LLAMA_FINAL_NORM = 0, 1, 2
LLAMA_ATTN_NORM, LLAMA_FFN_NORM, LLAMA_W_QKV, LLAMA_W_O = 10, 11, 12, 13
LLAMA_W_GATE_UP, LLAMA_W_DOWN, LLAMA_POOL_K, LLAMA_POOL_V = 14, 15, 16, 17


class LlamaModel:
    """The C ABI model runner: prefill_gpu / decode_step_gpu / on-device
    greedy generation (host buffers are numpy arrays)."""

    def __init__(self, config: LlamaConfig, seed: int, max_ctx: int):
        import numpy as np
        self._np = np
        self.config = config
        self.max_ctx = max_ctx
        h = ctypes.c_void_p()
        _check(load().kvhp_llama_create(ctypes.byref(config), seed, max_ctx, ctypes.byref(h)))
        self._h = h

    def close(self):
        if self._h:
            load().kvhp_llama_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def prefill(self, tokens):
        np = self._np
        t = np.ascontiguousarray(tokens, np.int32)
        logits = np.empty(self.config.vocab_size, np.float32)
        nxt = ctypes.c_int32()
        _check(load().kvhp_llama_prefill(self._h, t.ctypes.data, t.size, logits.ctypes.data,
                                         ctypes.byref(nxt)))
        return int(nxt.value), logits

    def decode_step(self, token: int = -1):
        np = self._np
        logits = np.empty(self.config.vocab_size, np.float32)
        nxt = ctypes.c_int32()
        _check(load().kvhp_llama_decode_step(self._h, token, logits.ctypes.data,
                                             ctypes.byref(nxt)))
        return int(nxt.value), logits

    def generate(self, n_steps: int, use_graph: bool = True):
        """Returns (tokens since the prefill, device milliseconds of the steps)."""
        np = self._np
        out = np.zeros(self.max_ctx + 1, np.int32)
        ms = ctypes.c_float()
        _check(load().kvhp_llama_generate(self._h, n_steps, int(use_graph), out.ctypes.data,
                                          ctypes.byref(ms)))
        return out, float(ms.value)

    def prefill_paged(self, tokens, pool, num_pages: int, block_table, max_pages: int,
                      stream=None):
        """Runner.prefill over a caller-owned pool [L][2][Hkv][num_pages][16][D]
        (torch fp16) and one block-table row (torch int32, device): returns
        (first greedy token, fp32 logits of the last position)."""
        np = self._np
        t = np.ascontiguousarray(tokens, np.int32)
        logits = np.empty(self.config.vocab_size, np.float32)
        nxt = ctypes.c_int32()
        _check(load().kvhp_llama_prefill_paged(self._h, t.ctypes.data, t.size, _ptr(pool),
                                               num_pages, _ptr(block_table), max_pages,
                                               logits.ctypes.data, ctypes.byref(nxt),
                                               _stream(stream)))
        return int(nxt.value), logits

    def prefill_cached(self, tokens, num_cached: int, pool, num_pages: int, block_table,
                       max_pages: int, write_table=None, stream=None):
        """Runner.prefill in the "full" prefix mode: the first num_cached
        positions' K/V are already in the pages; only the rest is forwarded
        (appends through write_table if given)."""
        np = self._np
        t = np.ascontiguousarray(tokens, np.int32)
        logits = np.empty(self.config.vocab_size, np.float32)
        nxt = ctypes.c_int32()
        _check(load().kvhp_llama_prefill_cached(self._h, t.ctypes.data, t.size, num_cached,
                                                _ptr(pool), num_pages, _ptr(block_table),
                                                _ptr(write_table), max_pages, logits.ctypes.data,
                                                ctypes.byref(nxt), _stream(stream)))
        return int(nxt.value), logits

    def decode_paged(self, tokens, pool, num_pages: int, block_tables, max_pages: int, positions,
                     seq_lens, max_seq_len: int, logits, next_tokens, stream=None):
        """Runner.decode_step for tokens.numel() sequences; every argument is a
        device tensor (int32, fp16 pool, fp32 logits [B][V]); asynchronous."""
        _check(load().kvhp_llama_decode_paged(self._h, _ptr(tokens), tokens.numel(), _ptr(pool),
                                              num_pages, _ptr(block_tables), max_pages,
                                              _ptr(positions), _ptr(seq_lens), max_seq_len,
                                              _ptr(logits), _ptr(next_tokens), _stream(stream)))

    def reserve(self, max_batch: int, max_seq_len: int):
        """Size the decode buffers for every decode_paged call up to these
        limits (required before capturing decode_paged in a HIP graph)."""
        _check(load().kvhp_llama_reserve(self._h, max_batch, max_seq_len))

    def tensor(self, layer: int, which: int):
        """Host copy (numpy float16) of a model tensor."""
        np = self._np
        ptr = ctypes.c_void_p()
        n = ctypes.c_size_t()
        _check(load().kvhp_llama_tensor(self._h, layer, which, ctypes.byref(ptr), ctypes.byref(n)))
        out = np.empty(n.value, np.float16)
        hip = ctypes.CDLL("libamdhip64.so")
        hip.hipMemcpy.argtypes = [_vp, _vp, _sz, _i32]
        hip.hipMemcpy.restype = _i32
        rc = hip.hipMemcpy(out.ctypes.data, ptr.value, n.value * 2, 2)  # device to host
        if rc != 0:
            raise KVHPError(KVHP_ERR_HIP, f"hipMemcpy device-to-host failed ({rc})")
        return out

    def set_tensor(self, layer: int, which: int, values):
        """Overwrite a model tensor from a host array of its element count
        (synchronous).  Batched decode steps see the new weights after the
        next reserve(), which rebuilds their tiled copies."""
        np = self._np
        ptr = ctypes.c_void_p()
        n = ctypes.c_size_t()
        _check(load().kvhp_llama_tensor(self._h, layer, which, ctypes.byref(ptr), ctypes.byref(n)))
        src = np.ascontiguousarray(values, np.float16).reshape(-1)
        if src.size != n.value:
            raise KVHPError(KVHP_ERR_INVALID, f"tensor holds {n.value} elements, got {src.size}")
        hip = ctypes.CDLL("libamdhip64.so")
        hip.hipMemcpy.argtypes = [_vp, _vp, _sz, _i32]
        hip.hipMemcpy.restype = _i32
        rc = hip.hipMemcpy(ptr.value, src.ctypes.data, src.size * 2, 1)  # host to device
        if rc != 0:
            raise KVHPError(KVHP_ERR_HIP, f"hipMemcpy host-to-device failed ({rc})")
