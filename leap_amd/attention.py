"""Python binding of the C-ABI in include/leap_hip_attention.h.

``HipAttention`` owns one library handle: the device key/value caches in the
reference engine's layout and the RoPE table.  Its methods map one-to-one to
the C entry points and raise ``LeapError`` on a negative status, the way the
reference engine raises ``std::runtime_error`` around its layer step.

Host arrays are numpy float32; the ``*_async`` methods take raw device
addresses (integers, e.g. ``tensor.data_ptr()``) and a raw ``hipStream_t``
(``torch.cuda.Stream().cuda_stream``), so torch is plumbing only.
"""
from __future__ import annotations

import ctypes
import errno
import os

import numpy as np

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libleap_hip_attention.so")
# the timeline build (the same sources compiled with LEAP_TIMELINE): decode
# launches record per-workgroup device-clock stamps (leap_hip_attention_timeline)
LIB_TL_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libleap_hip_attention_tl.so")

_F = ctypes.POINTER(ctypes.c_float)
_I = ctypes.c_int
_P = ctypes.c_void_p
_B = ctypes.POINTER(ctypes.c_int8)

EXPORTS = (
    "leap_hip_attention_create", "leap_hip_attention_destroy", "leap_hip_attention_last_error",
    "leap_hip_attention_step", "leap_hip_attention_step_async",
    "leap_hip_attention_step_batched", "leap_hip_attention_step_batched_async",
    "leap_hip_attention_clear", "leap_hip_attention_kv_upload", "leap_hip_attention_kv_download",
    "leap_hip_attention_kv_fill_normal", "leap_hip_attention_rope_download",
    "leap_hip_attention_set_split", "leap_hip_attention_kv_device_ptr",
    "leap_hip_attention_set_layer_weights", "leap_hip_attention_block",
    "leap_hip_attention_block_async", "leap_hip_attention_set_layer_weights_q8",
    "leap_hip_attention_block_views_get", "leap_hip_attention_checkpoint_read",
    "leap_hip_attention_load_checkpoint", "leap_hip_attention_packet_header",
    "leap_hip_attention_packet_upload", "leap_hip_attention_packet_download",
    "leap_hip_attention_xcc_map", "leap_hip_attention_step_noalloc", "leap_hip_attention_floor_async",
    "leap_hip_attention_set_products", "leap_hip_attention_set_fold_helper", "leap_hip_attention_timeline",
    "leap_hip_attention_create_q8kv", "leap_hip_attention_prompt", "leap_hip_attention_prompt_async",
    "leap_hip_attention_tree", "leap_hip_attention_tree_async", "leap_hip_attention_tree_keep",
    "leap_hip_attention_tree_keep_async", "leap_hip_attention_kv_write_async", "leap_hip_attention_kv_read_async",
    "leap_hip_attention_kv_q8_device_ptr",
    "leap_hip_attention_pages_create", "leap_hip_attention_pages_destroy", "leap_hip_attention_pages_last_error",
    "leap_hip_attention_pages_reserve", "leap_hip_attention_pages_reserve_async", "leap_hip_attention_pages_fork",
    "leap_hip_attention_pages_fork_async", "leap_hip_attention_pages_compact", "leap_hip_attention_pages_compact_async",
    "leap_hip_attention_pages_step", "leap_hip_attention_pages_step_async", "leap_hip_attention_pages_step_sparse",
    "leap_hip_attention_pages_step_sparse_async", "leap_hip_attention_pages_write", "leap_hip_attention_pages_write_async",
    "leap_hip_attention_pages_read", "leap_hip_attention_pages_read_async", "leap_hip_attention_pages_clear",
    "leap_hip_attention_pages_state", "leap_hip_attention_pages_view", "leap_hip_attention_pages_beam_select",
    "leap_hip_attention_pages_beam_select_async",
)

PACKET_HEADER_BYTES = 8
FLAG_NO_REPLY, FLAG_NEED_REPLY = 0, 1


class Checkpoint(ctypes.Structure):
    """leap_hip_attention_checkpoint: a checkpoint file's header."""
    _fields_ = [(n, ctypes.c_int) for n in ("version", "dim", "hidden_dim", "n_layers", "n_heads", "n_kv_heads",
                                            "vocab_size", "seq_len", "shared_classifier", "group_size")] + \
               [(n, ctypes.c_longlong) for n in ("header_bytes", "attention_bytes", "file_bytes")]


class BlockViews(ctypes.Structure):
    """leap_hip_attention_block_views: device addresses of the sub-block's
    intermediates after the last block call."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "att", "xq", "xs", "aq", "as_")]


class LeapError(RuntimeError):
    def __init__(self, code: int, msg: str):
        name = errno.errorcode.get(-code, str(code))
        super().__init__(f"{msg} ({name})")
        self.code = code


class Config(ctypes.Structure):
    _fields_ = [
        ("n_layers", _I), ("layer_begin", _I), ("layer_end", _I), ("n_heads", _I),
        ("n_kv_heads", _I), ("head_dim", _I), ("seq_len", _I), ("rope_theta", ctypes.c_float),
        ("max_batch", _I), ("device", _I),
    ]


class PagesConfig(ctypes.Structure):
    _fields_ = [("model", Config), ("page_rows", _I), ("n_pages", _I), ("q8", _I), ("bounds", _I)]


class PagesArrays(ctypes.Structure):
    """leap_hip_attention_pages_arrays: device addresses of a layer's pages and of the table."""
    _fields_ = [("table", _P), ("refs", _P), ("width", _I)] + [(n, _P) for n in ("k", "v", "ks", "vs", "bounds")]


_lib = None
_lib_tl = None


def load_library(path: str = LIB_PATH):
    """Load the HIP library; fails loudly when it has not been built."""
    global _lib
    if _lib is None:
        _lib = _open(path)
    return _lib


def load_timeline_library():
    """Load the timeline build of the library (its own copy of every entry
    point, with leap_hip_attention_timeline recording); handles made with it
    are passed `lib=` this library."""
    global _lib_tl
    if _lib_tl is None:
        _lib_tl = _open(LIB_TL_PATH)
    return _lib_tl


def _open(path: str):
    if not os.path.isfile(path):
        raise RuntimeError(f"{path} is missing: build it with `python -m leap_amd.build`")
    L = ctypes.CDLL(path)
    H = _P
    L.leap_hip_attention_create.argtypes = [ctypes.POINTER(Config), ctypes.POINTER(H)]
    L.leap_hip_attention_destroy.argtypes = [H]
    L.leap_hip_attention_last_error.argtypes = [H]
    L.leap_hip_attention_last_error.restype = ctypes.c_char_p
    L.leap_hip_attention_step.argtypes = [H, _I, _I, _F, _F, _F, _F]
    L.leap_hip_attention_step_async.argtypes = [H, _I, _I, _P, _P, _P, _P, _P]
    L.leap_hip_attention_step_batched.argtypes = [H, _I, _I, ctypes.POINTER(_I), _F, _F, _F, _F]
    L.leap_hip_attention_step_batched_async.argtypes = [H, _I, _I, _P, _I, ctypes.c_longlong, _P, _P,
                                                        _P, _P, _P]
    L.leap_hip_attention_clear.argtypes = [H]
    L.leap_hip_attention_kv_upload.argtypes = [H, _I, _I, _I, _I, _F, _F]
    L.leap_hip_attention_kv_download.argtypes = [H, _I, _I, _I, _I, _F, _F]
    L.leap_hip_attention_kv_fill_normal.argtypes = [H, ctypes.c_uint64, ctypes.c_float]
    L.leap_hip_attention_rope_download.argtypes = [H, _I, _I, _F, _F]
    L.leap_hip_attention_set_split.argtypes = [H, _I]
    L.leap_hip_attention_kv_device_ptr.argtypes = [H, _I, _I, ctypes.POINTER(_P),
                                                   ctypes.POINTER(_P)]
    L.leap_hip_attention_set_layer_weights.argtypes = [H, _I, _F, _F, _F, _F, _F]
    L.leap_hip_attention_block.argtypes = [H, _I, _I, _F]
    L.leap_hip_attention_block_async.argtypes = [H, _I, _I, _P, _P]
    L.leap_hip_attention_set_layer_weights_q8.argtypes = [H, _I, _I, _F] + [_B, _F] * 4
    L.leap_hip_attention_block_views_get.argtypes = [H, ctypes.POINTER(BlockViews)]
    L.leap_hip_attention_checkpoint_read.argtypes = [ctypes.c_char_p, ctypes.POINTER(Checkpoint)]
    L.leap_hip_attention_load_checkpoint.argtypes = [H, ctypes.c_char_p]
    _IP = ctypes.POINTER(_I)
    L.leap_hip_attention_packet_header.argtypes = [ctypes.c_char_p, ctypes.c_size_t, _I, _IP, _IP]
    L.leap_hip_attention_packet_upload.argtypes = [H, ctypes.c_char_p, ctypes.c_size_t, _P, _IP, _IP, _P]
    L.leap_hip_attention_packet_download.argtypes = [H, _P, _I, _I, _P, ctypes.c_size_t, _P]
    L.leap_hip_attention_xcc_map.argtypes = [_I, _I, ctypes.POINTER(_I)]
    L.leap_hip_attention_floor_async.argtypes = [H, _I, _I, _I, _P, _I, ctypes.c_longlong, _P]
    L.leap_hip_attention_set_products.argtypes = [H, _I]
    L.leap_hip_attention_set_fold_helper.argtypes = [H, _I]
    L.leap_hip_attention_step_noalloc.argtypes = [ctypes.POINTER(Config), _I] + [_P] * 8
    L.leap_hip_attention_create_q8kv.argtypes = [ctypes.POINTER(Config), ctypes.POINTER(H)]
    L.leap_hip_attention_prompt.argtypes = [H, _I, _I, _IP, _IP, _F, _F, _F, _F]
    L.leap_hip_attention_prompt_async.argtypes = [H, _I, _I, _P, _P, _I, _I, _I, _P, _P, _P, _P, _P]
    L.leap_hip_attention_tree.argtypes = [H, _I, _I, _IP, _IP, _IP, _F, _F, _F, _F]
    L.leap_hip_attention_tree_async.argtypes = [H, _I, _I, _P, _P, _P, _I, _I, _I, _P, _P, _P, _P, _P]
    L.leap_hip_attention_tree_keep.argtypes = [H, _I, _IP, _IP, _I]
    L.leap_hip_attention_tree_keep_async.argtypes = [H, _I, _P, _P, _I, _P]
    L.leap_hip_attention_kv_write_async.argtypes = [H, _I, _I, _I, _I, _P, _P, _P]
    L.leap_hip_attention_kv_read_async.argtypes = [H, _I, _I, _I, _I, _P, _P, _P]
    L.leap_hip_attention_kv_q8_device_ptr.argtypes = [H, _I, _I] + [ctypes.POINTER(_P)] * 4
    L.leap_hip_attention_timeline.argtypes = [_P, ctypes.c_size_t, ctypes.POINTER(ctypes.c_longlong)]
    pages = {
        "create": [ctypes.POINTER(PagesConfig), ctypes.POINTER(H)], "destroy": [H], "last_error": [H], "clear": [H],
        "reserve": [H, _I, _IP, _IP], "reserve_async": [H, _I, _P, _P, _P, _P],
        "fork": [H, _I, _IP, _IP], "fork_async": [H, _I, _P, _P, _P],
        "compact": [H, _IP], "compact_async": [H, _P, _P],
        "step": [H, _I, _I, _IP, _F, _F, _F, _F],
        "step_async": [H, _I, _I, _P, _I, ctypes.c_longlong] + [_P] * 5,
        "step_sparse": [H, _I, _I, _IP, _I, _F, _F, _F, _F, _IP],
        "step_sparse_async": [H, _I, _I, _P, _I, _I] + [_P] * 6,
        "write": [H, _I, _I, _I, _I, _F, _F], "write_async": [H, _I, _I, _I, _I, _P, _P, _P],
        "read": [H, _I, _I, _I, _I, _F, _F], "read_async": [H, _I, _I, _I, _I, _P, _P, _P],
        "state": [H, _IP, _IP], "view": [H, _I, ctypes.POINTER(PagesArrays)],
        "beam_select": [H, _I, _I, _I, _F, _F, _IP, _IP, _F],
        "beam_select_async": [H, _I, _I, _I, _P, ctypes.c_longlong] + [_P] * 5,
    }
    for name, types in pages.items():
        getattr(L, "leap_hip_attention_pages_" + name).argtypes = types
    L.leap_hip_attention_pages_last_error.restype = ctypes.c_char_p
    for name in EXPORTS:
        fn = getattr(L, name)
        if not name.endswith("_last_error"):
            fn.restype = _I
    return L


def _fp(a):
    if a is None:
        return None
    assert a.dtype == np.float32 and a.flags.c_contiguous
    return a.ctypes.data_as(_F)


def _i32(a):
    return np.ascontiguousarray(a, dtype=np.int32).reshape(-1)


def _ip(a):
    return a.ctypes.data_as(ctypes.POINTER(_I))


def _f32(a, n=None):
    a = np.ascontiguousarray(a, dtype=np.float32).reshape(-1)
    if n is not None and a.size != n:
        raise ValueError(f"expected {n} floats, got {a.size}")
    return a


def checkpoint_read(path) -> dict:
    """The header of a LEAP checkpoint file (no GPU needed)."""
    lib = load_library()
    c = Checkpoint()
    rc = lib.leap_hip_attention_checkpoint_read(os.fsencode(path), ctypes.byref(c))
    if rc != 0:
        raise LeapError(rc, f"{path}: {'cannot read' if rc == -errno.EIO else 'not a LEAP checkpoint'}")
    return {n: getattr(c, n) for n, _ in Checkpoint._fields_}


def xcc_map(n_wg: int, device: int = 0) -> np.ndarray:
    """The XCD each of n_wg workgroups of the decode kernel's size ran on."""
    lib = load_library()
    out = np.empty(n_wg, np.int32)
    rc = lib.leap_hip_attention_xcc_map(device, n_wg, out.ctypes.data_as(ctypes.POINTER(_I)))
    if rc != 0:
        raise LeapError(rc, lib.leap_hip_attention_last_error(None).decode())
    return out


def step_noalloc(n_heads, n_kv_heads, head_dim, seq_len, pos, rope_ptr, k_cache_ptr, v_cache_ptr, q_ptr,
                 k_ptr, v_ptr, out_ptr, stream=0, device=0):
    """leap_hip_attention_step_noalloc on caller-owned device buffers (raw
    addresses): no handle and no device allocation."""
    lib = load_library()
    cfg = Config(1, 0, 1, n_heads, n_kv_heads, head_dim, seq_len, 0.0, 1, device)
    rc = lib.leap_hip_attention_step_noalloc(ctypes.byref(cfg), pos, rope_ptr, k_cache_ptr, v_cache_ptr, q_ptr,
                                             k_ptr, v_ptr, out_ptr, stream)
    if rc != 0:
        raise LeapError(rc, lib.leap_hip_attention_last_error(None).decode())


def packet_header(packet: bytes, dim):
    """(pos, flags) of a stage packet, or None for a control packet (no GPU needed)."""
    pos, flags = _I(), _I()
    rc = load_library().leap_hip_attention_packet_header(packet, len(packet), dim, ctypes.byref(pos),
                                                         ctypes.byref(flags))
    if rc < 0:
        raise LeapError(rc, f"packet of {len(packet)} bytes is not 8 + 4*{dim}")
    return None if rc == 1 else (pos.value, flags.value)


class HipAttention:
    """One handle of the MI355X attention library (see the C header).
    cache: "f32", the engine's cache, or "q8", int8 values with a scale per
    row and KV head."""

    def __init__(self, n_heads, n_kv_heads, head_dim, seq_len, n_layers=1, layer_begin=0,
                 layer_end=None, rope_theta=500000.0, max_batch=1, device=0, lib=None, cache="f32"):
        if cache not in ("f32", "q8"):
            raise ValueError(f"cache {cache!r} is not 'f32' or 'q8'")
        self.lib = lib if lib is not None else load_library()
        self.cfg = Config(n_layers, layer_begin, n_layers if layer_end is None else layer_end,
                          n_heads, n_kv_heads, head_dim, seq_len, rope_theta, max_batch, device)
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.seq_len, self.max_batch = seq_len, max_batch
        self.q_dim, self.kv_dim = n_heads * head_dim, n_kv_heads * head_dim
        h = _P()
        create = self.lib.leap_hip_attention_create_q8kv if cache == "q8" else self.lib.leap_hip_attention_create
        rc = create(ctypes.byref(self.cfg), ctypes.byref(h))
        if rc != 0:
            raise LeapError(rc, self.lib.leap_hip_attention_last_error(None).decode())
        self.h = h

    # -- lifetime -----------------------------------------------------------
    def close(self):
        if getattr(self, "h", None):
            self.lib.leap_hip_attention_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        if rc != 0:
            raise LeapError(rc, self.lib.leap_hip_attention_last_error(self.h).decode())

    # -- the step -----------------------------------------------------------
    def step(self, layer, pos, q, k_new, v_new):
        q, k, v = _f32(q, self.q_dim), _f32(k_new, self.kv_dim), _f32(v_new, self.kv_dim)
        out = np.empty(self.q_dim, np.float32)
        self._check(self.lib.leap_hip_attention_step(self.h, layer, pos, _fp(q), _fp(k), _fp(v),
                                                     _fp(out)))
        return out

    def step_async(self, layer, pos, q_ptr, k_ptr, v_ptr, out_ptr, stream=0):
        self._check(self.lib.leap_hip_attention_step_async(self.h, layer, pos, q_ptr, k_ptr,
                                                           v_ptr, out_ptr, stream))

    def step_batched(self, layer, pos, q, k_new, v_new):
        pos = np.ascontiguousarray(pos, dtype=np.int32).reshape(-1)
        n = pos.size
        q = _f32(q, n * self.q_dim)
        k, v = _f32(k_new, n * self.kv_dim), _f32(v_new, n * self.kv_dim)
        out = np.empty(n * self.q_dim, np.float32)
        self._check(self.lib.leap_hip_attention_step_batched(
            self.h, layer, n, pos.ctypes.data_as(ctypes.POINTER(_I)), _fp(q), _fp(k), _fp(v),
            _fp(out)))
        return out.reshape(n, self.q_dim)

    def step_batched_async(self, layer, n_seq, pos_ptr, max_pos, q_ptr, k_ptr, v_ptr, out_ptr,
                           stream=0, total_rows=0):
        """total_rows: sum of pos[i] + 1 if known on the host (sizes the split), else 0."""
        self._check(self.lib.leap_hip_attention_step_batched_async(
            self.h, layer, n_seq, pos_ptr, max_pos, total_rows, q_ptr, k_ptr, v_ptr, out_ptr,
            stream))

    # -- several tokens of each sequence ------------------------------------
    def _many_in(self, begin, pos, q, k_new, v_new):
        begin, pos = _i32(begin), _i32(pos)
        if begin.size != pos.size + 1:
            raise ValueError(f"{pos.size} positions need {pos.size + 1} begins, got {begin.size}")
        n = max(0, int(begin[-1]))
        return begin, pos, n, _f32(q, n * self.q_dim), _f32(k_new, n * self.kv_dim), _f32(v_new, n * self.kv_dim)

    def prompt(self, layer, begin, pos, q, k_new, v_new):
        """New tokens of each sequence, causal over its cache: sequence i has the rows
        begin[i]:begin[i + 1] of q, k_new and v_new, from position pos[i] on.  Rows ahead
        of begin[0] come back as zeros."""
        begin, pos, n, q, k, v = self._many_in(begin, pos, q, k_new, v_new)
        out = np.zeros(n * self.q_dim, np.float32)
        self._check(self.lib.leap_hip_attention_prompt(self.h, layer, pos.size, _ip(begin), _ip(pos), _fp(q), _fp(k),
                                                       _fp(v), _fp(out)))
        return out.reshape(n, self.q_dim)

    def prompt_async(self, layer, n_seq, begin_ptr, pos_ptr, n_tokens, max_tokens, max_pos, q_ptr, k_ptr, v_ptr,
                     out_ptr, stream=0):
        """n_tokens: rows of the packed arrays; max_tokens, max_pos: upper bounds of a
        sequence's tokens and of the positions they take."""
        self._check(self.lib.leap_hip_attention_prompt_async(
            self.h, layer, n_seq, begin_ptr, pos_ptr, n_tokens, max_tokens, max_pos, q_ptr, k_ptr, v_ptr, out_ptr,
            stream))

    def tree(self, layer, begin, pos, parent, q, k_new, v_new):
        """A tree of drafted tokens of each sequence: node j (row begin[i] + j) hangs on
        node parent[begin[i] + j] < j, or on the cached rows (-1)."""
        begin, pos, n, q, k, v = self._many_in(begin, pos, q, k_new, v_new)
        parent = _i32(parent)
        if parent.size != n:
            raise ValueError(f"expected {n} parents, got {parent.size}")
        out = np.zeros(n * self.q_dim, np.float32)
        self._check(self.lib.leap_hip_attention_tree(self.h, layer, pos.size, _ip(begin), _ip(pos), _ip(parent), _fp(q),
                                                     _fp(k), _fp(v), _fp(out)))
        return out.reshape(n, self.q_dim)

    def tree_async(self, layer, n_seq, begin_ptr, pos_ptr, parent_ptr, n_tokens, max_tokens, max_pos, q_ptr, k_ptr,
                   v_ptr, out_ptr, stream=0):
        self._check(self.lib.leap_hip_attention_tree_async(
            self.h, layer, n_seq, begin_ptr, pos_ptr, parent_ptr, n_tokens, max_tokens, max_pos, q_ptr, k_ptr, v_ptr,
            out_ptr, stream))

    def tree_keep(self, pos, path):
        """Move the rows of each sequence's accepted nodes path[i] (ascending, ended by
        -1) to the rows from pos[i] on, in every held layer."""
        pos = _i32(pos)
        path = np.ascontiguousarray(path, np.int32).reshape(pos.size, -1)
        self._check(self.lib.leap_hip_attention_tree_keep(self.h, pos.size, _ip(pos), _ip(path), path.shape[1]))

    def tree_keep_async(self, n_seq, pos_ptr, path_ptr, max_path, stream=0):
        self._check(self.lib.leap_hip_attention_tree_keep_async(self.h, n_seq, pos_ptr, path_ptr, max_path, stream))

    # -- the attention sub-block (rmsnorm, q/k/v, attention, wo, residual) ---
    def set_layer_weights(self, layer, rms_att, wq, wk, wv, wo):
        """Upload one layer's weights, row-major as the reference holds them."""
        d, kv = self.q_dim, self.kv_dim
        arrs = (_f32(rms_att, d), _f32(wq, d * d), _f32(wk, kv * d), _f32(wv, kv * d), _f32(wo, d * d))
        self._check(self.lib.leap_hip_attention_set_layer_weights(self.h, layer, *(_fp(a) for a in arrs)))

    def set_layer_weights_q8(self, layer, group_size, rms_att, wq, wk, wv, wo):
        """Upload one layer's int8 weights: each of wq, wk, wv, wo is (int8
        values [d][n], float scales [d*n/group_size]) as the quantized engine
        holds them."""
        d, kv = self.q_dim, self.kv_dim
        arrs = [_f32(rms_att, d)]  # held here until the upload returns
        for (q, sc), rows in ((wq, d), (wk, kv), (wv, kv), (wo, d)):
            q = np.ascontiguousarray(q, np.int8).reshape(-1)
            if q.size != rows * d:
                raise ValueError(f"expected {rows * d} int8 values, got {q.size}")
            arrs += [q, _f32(sc, rows * d // group_size)]
        args = [a.ctypes.data_as(_B) if a.dtype == np.int8 else _fp(a) for a in arrs]
        self._check(self.lib.leap_hip_attention_set_layer_weights_q8(self.h, layer, group_size, *args))

    def load_checkpoint(self, path):
        """Upload every held layer's attention weights from a checkpoint file."""
        self._check(self.lib.leap_hip_attention_load_checkpoint(self.h, os.fsencode(path)))

    def block_views(self) -> dict:
        """Device addresses of the last block call's intermediates
        (q, k, v, att; xq, xs, aq, as_ with int8 weights, else None)."""
        bv = BlockViews()
        self._check(self.lib.leap_hip_attention_block_views_get(self.h, ctypes.byref(bv)))
        return {n: getattr(bv, n) for n, _ in BlockViews._fields_}

    def block(self, layer, pos, x):
        """x + Wo . attention(Wq/Wk/Wv . rmsnorm(x)); returns the new residual stream."""
        x = _f32(x, self.q_dim).copy()
        self._check(self.lib.leap_hip_attention_block(self.h, layer, pos, _fp(x)))
        return x

    def block_async(self, layer, pos, x_ptr, stream=0):
        self._check(self.lib.leap_hip_attention_block_async(self.h, layer, pos, x_ptr, stream))

    # -- stage hand-off -----------------------------------------------------
    def packet_upload(self, packet: bytes, x_ptr, stream=0):
        """Copy a data packet's x to device memory at x_ptr; returns (pos, flags),
        or None for a control packet.  stream 0: synchronous."""
        pos, flags = _I(), _I()
        rc = self.lib.leap_hip_attention_packet_upload(self.h, packet, len(packet), x_ptr, ctypes.byref(pos),
                                                       ctypes.byref(flags), stream)
        if rc == 1:
            return None
        self._check(rc)
        return pos.value, flags.value

    def packet_download(self, x_ptr, pos, flags) -> bytes:
        """The packet {pos, flags} + x (device memory at x_ptr), synchronously."""
        buf = ctypes.create_string_buffer(PACKET_HEADER_BYTES + 4 * self.q_dim)
        self._check(self.lib.leap_hip_attention_packet_download(self.h, x_ptr, pos, flags, buf, len(buf), None))
        return buf.raw

    # -- cache management ---------------------------------------------------
    def clear(self):
        self._check(self.lib.leap_hip_attention_clear(self.h))

    def kv_upload(self, seq, layer, pos_begin, k=None, v=None):
        rows = None
        if k is not None:
            k = _f32(k)
            rows = k.size // self.kv_dim
        if v is not None:
            v = _f32(v)
            rows = v.size // self.kv_dim if rows is None else rows
        if rows is None:
            return
        self._check(self.lib.leap_hip_attention_kv_upload(self.h, seq, layer, pos_begin,
                                                          pos_begin + rows, _fp(k), _fp(v)))

    def kv_download(self, seq, layer, pos_begin, pos_end):
        k = np.empty((pos_end - pos_begin, self.kv_dim), np.float32)
        v = np.empty_like(k)
        self._check(self.lib.leap_hip_attention_kv_download(self.h, seq, layer, pos_begin,
                                                            pos_end, _fp(k), _fp(v)))
        return k, v

    def kv_write_async(self, seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream=0):
        """fp32 rows in device memory into the cache (an 8-bit one: quantised); either may be 0."""
        self._check(self.lib.leap_hip_attention_kv_write_async(self.h, seq, layer, pos_begin, pos_end, k_ptr, v_ptr,
                                                               stream))

    def kv_read_async(self, seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream=0):
        """The cache's rows as fp32 into device memory; either may be 0."""
        self._check(self.lib.leap_hip_attention_kv_read_async(self.h, seq, layer, pos_begin, pos_end, k_ptr, v_ptr,
                                                              stream))

    def kv_q8_device_ptr(self, seq, layer):
        """Device addresses of an 8-bit cache: key values and scales, value values and scales."""
        p = [_P() for _ in range(4)]
        self._check(self.lib.leap_hip_attention_kv_q8_device_ptr(self.h, seq, layer, *(ctypes.byref(x) for x in p)))
        return tuple(x.value for x in p)

    def kv_fill_normal(self, seed, scale):
        self._check(self.lib.leap_hip_attention_kv_fill_normal(self.h, seed, scale))

    def rope_download(self, pos_begin=0, pos_end=None):
        pos_end = self.seq_len if pos_end is None else pos_end
        c = np.empty((pos_end - pos_begin, self.head_dim // 2), np.float32)
        s = np.empty_like(c)
        self._check(self.lib.leap_hip_attention_rope_download(self.h, pos_begin, pos_end,
                                                              _fp(c), _fp(s)))
        return c, s

    def floor_async(self, kind, layer, n_seq, max_pos, total_rows, stream=0, pos_ptr=None):
        """Enqueue a floor launch of a step's shape: kind 1 launch only,
        kind 2 the bare K/V stream (measurement; writes nothing).  pos_ptr:
        device address of the n_seq positions, or None for every sequence
        at max_pos."""
        self._check(self.lib.leap_hip_attention_floor_async(self.h, kind, layer, n_seq, pos_ptr, max_pos,
                                                            total_rows, stream))

    def set_products(self, valu: bool):
        """Score and weighted-V products on the VALU (True) or the matrix cores."""
        self._check(self.lib.leap_hip_attention_set_products(self.h, 1 if valu else 0))

    def set_fold_helper(self, mode: int):
        """How a one-level merge's final fold is shared: 1 two workgroups (the
        default), 0 the last workgroup alone, 2 the fallback path (the helper
        gives up at once)."""
        self._check(self.lib.leap_hip_attention_set_fold_helper(self.h, mode))

    def set_split(self, chunk_positions):
        self._check(self.lib.leap_hip_attention_set_split(self.h, chunk_positions))

    def kv_device_ptr(self, seq, layer):
        k, v = _P(), _P()
        self._check(self.lib.leap_hip_attention_kv_device_ptr(self.h, seq, layer,
                                                              ctypes.byref(k), ctypes.byref(v)))
        return k.value, v.value


class PagedAttention:
    """One handle of a cache of pages (see the C header): sequences 0..max_batch-1 whose
    rows lie in pages of page_rows rows of a pool of n_pages.
    cache: "f32" or "q8"; bounds: keep what step_sparse chooses pages by."""

    def __init__(self, n_heads, n_kv_heads, head_dim, seq_len, n_pages, page_rows=16, n_layers=1, layer_begin=0,
                 layer_end=None, rope_theta=500000.0, max_batch=1, device=0, cache="f32", bounds=False):
        if cache not in ("f32", "q8"):
            raise ValueError(f"cache {cache!r} is not 'f32' or 'q8'")
        self.lib = load_library()
        model = Config(n_layers, layer_begin, n_layers if layer_end is None else layer_end, n_heads, n_kv_heads, head_dim,
                       seq_len, rope_theta, max_batch, device)
        self.cfg = PagesConfig(model, page_rows, n_pages, cache == "q8", bool(bounds))
        self.n_kv_heads, self.max_batch, self.n_pages, self.seq_len = n_kv_heads, max_batch, n_pages, seq_len
        self.q_dim, self.kv_dim = n_heads * head_dim, n_kv_heads * head_dim
        self.width = -(-seq_len // page_rows) if page_rows > 0 else 0
        h = _P()
        rc = self.lib.leap_hip_attention_pages_create(ctypes.byref(self.cfg), ctypes.byref(h))
        if rc != 0:
            raise LeapError(rc, self.lib.leap_hip_attention_pages_last_error(None).decode())
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            self.lib.leap_hip_attention_pages_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _call(self, name, *args):
        rc = getattr(self.lib, "leap_hip_attention_pages_" + name)(self.h, *args)
        if rc != 0:
            raise LeapError(rc, self.lib.leap_hip_attention_pages_last_error(self.h).decode())

    @staticmethod
    def _pair(a, b, what):
        a, b = _i32(a), _i32(b)
        if a.size != b.size:
            raise ValueError(f"{what}: {a.size} and {b.size} values")
        return a, b

    # -- pages ----------------------------------------------------------------
    def reserve(self, begin, end):
        """Pages of its own for rows [begin[i], end[i]) of each sequence."""
        begin, end = self._pair(begin, end, "begin and end")
        self._call("reserve", begin.size, _ip(begin), _ip(end))

    def reserve_async(self, n_seq, begin_ptr, end_ptr, status_ptr=0, stream=0):
        self._call("reserve_async", n_seq, begin_ptr, end_ptr, status_ptr, stream)

    def fork(self, parent, rows):
        """Sequence i takes the pages of the first rows[i] rows of parent[i] (None: each its own)."""
        if parent is None:
            rows = _i32(rows)
            self._call("fork", rows.size, None, _ip(rows))
        else:
            parent, rows = self._pair(parent, rows, "parent and rows")
            self._call("fork", rows.size, _ip(parent), _ip(rows))

    def fork_async(self, n_seq, parent_ptr, rows_ptr, stream=0):
        self._call("fork_async", n_seq, parent_ptr, rows_ptr, stream)

    def compact(self):
        """The pages in use moved to the pool's front; how many they are."""
        used = _I()
        self._call("compact", ctypes.byref(used))
        return used.value

    def compact_async(self, used_ptr=0, stream=0):
        self._call("compact_async", used_ptr, stream)

    def state(self):
        """The table [max_batch][width] and the pages' numbers of references."""
        table, refs = np.empty((self.max_batch, self.width), np.int32), np.empty(self.n_pages, np.int32)
        self._call("state", _ip(table), _ip(refs))
        return table, refs

    def view(self, layer) -> dict:
        """Device addresses of the table, the references and a layer's pages (None where there are none)."""
        a = PagesArrays()
        self._call("view", layer, ctypes.byref(a))
        return {n: getattr(a, n) for n, _ in PagesArrays._fields_}

    def clear(self):
        self._call("clear")

    # -- the step ---------------------------------------------------------------
    def _step_in(self, pos, q, k_new, v_new):
        pos = _i32(pos)
        n = pos.size
        return pos, n, _f32(q, n * self.q_dim), _f32(k_new, n * self.kv_dim), _f32(v_new, n * self.kv_dim)

    def step(self, layer, pos, q, k_new, v_new):
        pos, n, q, k, v = self._step_in(pos, q, k_new, v_new)
        out = np.empty((n, self.q_dim), np.float32)
        self._call("step", layer, n, _ip(pos), _fp(q), _fp(k), _fp(v), _fp(out))
        return out

    def step_async(self, layer, n_seq, pos_ptr, max_pos, q_ptr, k_ptr, v_ptr, out_ptr, stream=0, total_rows=0):
        """total_rows: sum of pos[i] + 1 if known on the host (sizes and picks the launch), else 0."""
        self._call("step_async", layer, n_seq, pos_ptr, max_pos, total_rows, q_ptr, k_ptr, v_ptr, out_ptr, stream)

    def step_sparse(self, layer, pos, keep, q, k_new, v_new):
        """The step over at most `keep` pages a KV head; also returns which, [n_seq][n_kv_heads][keep]."""
        pos, n, q, k, v = self._step_in(pos, q, k_new, v_new)
        out = np.empty((n, self.q_dim), np.float32)
        picked = np.empty((n, self.n_kv_heads, max(keep, 1)), np.int32)
        self._call("step_sparse", layer, n, _ip(pos), keep, _fp(q), _fp(k), _fp(v), _fp(out), _ip(picked))
        return out, picked

    def step_sparse_async(self, layer, n_seq, pos_ptr, max_pos, keep, q_ptr, k_ptr, v_ptr, out_ptr, picked_ptr=0, stream=0):
        self._call("step_sparse_async", layer, n_seq, pos_ptr, max_pos, keep, q_ptr, k_ptr, v_ptr, out_ptr, picked_ptr, stream)

    # -- rows -------------------------------------------------------------------
    def write(self, seq, layer, pos_begin, k=None, v=None):
        k, v = (None if x is None else _f32(x) for x in (k, v))
        sizes = {x.size for x in (k, v) if x is not None}
        if len(sizes) > 1 or any(n % self.kv_dim for n in sizes):
            raise ValueError(f"k and v: {sorted(sizes)} values are no equal numbers of rows of {self.kv_dim}")
        rows = {n // self.kv_dim for n in sizes}
        if rows:
            self._call("write", seq, layer, pos_begin, pos_begin + rows.pop(), _fp(k), _fp(v))

    def write_async(self, seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream=0):
        self._call("write_async", seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream)

    def read(self, seq, layer, pos_begin, pos_end):
        k = np.empty((max(0, pos_end - pos_begin), self.kv_dim), np.float32)
        v = np.empty_like(k)
        self._call("read", seq, layer, pos_begin, pos_end, _fp(k), _fp(v))
        return k, v

    def read_async(self, seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream=0):
        self._call("read_async", seq, layer, pos_begin, pos_end, k_ptr, v_ptr, stream)

    # -- beams ------------------------------------------------------------------
    def beam_select(self, n_groups, beams, logits, score):
        """The best continuations of each group of beams: parent, token and score."""
        n = n_groups * beams
        logits = _f32(logits)
        vocab = logits.size // max(1, n)
        if logits.size != n * vocab:
            raise ValueError(f"{logits.size} logits of {n} beams")
        score = _f32(score, n)
        parent, token, best = np.empty(n, np.int32), np.empty(n, np.int32), np.empty(n, np.float32)
        self._call("beam_select", n_groups, beams, vocab, _fp(logits), _fp(score), _ip(parent), _ip(token), _fp(best))
        return parent, token, best

    def beam_select_async(self, n_groups, beams, vocab, logits_ptr, stride, score_ptr, parent_ptr, token_ptr, best_ptr, stream=0):
        self._call("beam_select_async", n_groups, beams, vocab, logits_ptr, stride, score_ptr, parent_ptr, token_ptr, best_ptr,
                   stream)
