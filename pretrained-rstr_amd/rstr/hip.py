"""ctypes binding of ``librstr_hip.so`` (declared in ``include/rstr_hip.h``).

This is the Python twin of the JDK 21 FFM binding a Clojure caller would use:
thin handles, plain int32/f32 arrays, negative status codes
turned into :class:`RstrError` carrying the library's message, the way the
reference raises ``ex-info``.  No computation happens here; every call goes to
the HIP library, and loading fails loudly if the library is missing.

The operators on device arrays (:class:`Kv4Pool`, :class:`Kv4Attention`,
:class:`Verifier`, :meth:`Session.step_maps`, and over the fp16 pages of a pool
:meth:`Pool.rope_append`, :class:`PagedAttention`, :class:`BlockBounds` and
:class:`BlockSelect`) take arrays that live on the
session's GPU: torch tensors, or anything with their ``data_ptr()``, ``shape``,
``stride()``, ``dtype`` and ``device``.  They queue work and return.  A program
that uses torch imports it before this library is loaded, so that both share
one HIP runtime.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import sys
import threading
import weakref

import numpy as np

PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG, "lib", "librstr_hip.so")

ROLE = dict(embed=0, final_norm=1, attn_norm=2, q=3, k=4, v=5, o=6, q_norm=7, k_norm=8,
            post_attn_norm=9, ffn_pre_norm=10, ffn_post_norm=11, gate=12, up=13, down=14)
KERNEL_CLASSES = ("qgemm", "head", "attn_split", "attn_merge", "qkv_post", "rows", "tail")

EXPORTS = (
    "rstr_session_open", "rstr_session_close", "rstr_last_error", "rstr_open_error",
    "rstr_session_memory",
    "rstr_model_bind", "rstr_model_bind_raw", "rstr_model_bind_synthetic", "rstr_model_close", "rstr_model_weight_bytes",
    "rstr_model_export_linear", "rstr_pool_open", "rstr_pool_close", "rstr_pool_copy_page",
    "rstr_pool_upload", "rstr_pool_download", "rstr_pool_fill_synthetic", "rstr_chunk_export_submit",
    "rstr_chunk_restore_submit", "rstr_transfer_done", "rstr_transfer_complete", "rstr_chunk_bench", "rstr_decoder_open",
    "rstr_decoder_close", "rstr_prime_lanes", "rstr_prime_rows", "rstr_step_lanes",
    "rstr_step_lanes_submit", "rstr_step_lanes_collect",
    "rstr_decode_logits", "rstr_decode_logits_device", "rstr_decoder_read_rows", "rstr_decoder_set_graph", "rstr_decoder_step_timing",
    "rstr_prefill_open",
    "rstr_prefill_range", "rstr_append_run", "rstr_tail_run", "rstr_linear_run",
    "rstr_attention_run", "rstr_attention_run_static",
    "rstr_attention_bench", "rstr_schedule_upload", "rstr_schedule_run",
    "rstr_decoder_profile_steps",
    "rstr_kv4_open", "rstr_kv4_close", "rstr_kv4_bytes", "rstr_kv4_append", "rstr_kv4_read",
    "rstr_kv4_attn_open", "rstr_kv4_attn_close", "rstr_kv4_attn_run",
    "rstr_step_maps", "rstr_verify_open", "rstr_verify_close", "rstr_verify_run",
    "rstr_pool_device", "rstr_pool_rope_append", "rstr_pool_attn_open", "rstr_pool_attn_close", "rstr_pool_attn_run",
    "rstr_bounds_open", "rstr_bounds_close", "rstr_bounds_device", "rstr_bounds_update", "rstr_select_open", "rstr_select_close", "rstr_select_run",
)


class RstrError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class Desc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "n_layers", "d_model", "d_ff", "n_q", "n_kv", "head_dim", "vocab", "weight_bits",
        "gain_offset", "qk_norm", "sandwich", "ffn_geglu", "rope_dual", "global_pattern",
        "sliding_window", "embed_scale_sqrt_d")] + [
        ("eps", C.c_float), ("attn_scale", C.c_float),
        ("rope_global", C.c_double), ("rope_local", C.c_double)]


class Tensor(C.Structure):
    _fields_ = [("layer", C.c_int32), ("role", C.c_int32), ("data", C.c_void_p),
                ("elements", C.c_int64)]


class RawTensor(C.Structure):
    _fields_ = [("layer", C.c_int32), ("role", C.c_int32), ("dtype", C.c_int32), ("data", C.c_void_p),
                ("elements", C.c_int64)]


RAW_DTYPES = {"F32": 0, "F16": 1, "BF16": 2}


class TransferStats(C.Structure):
    _fields_ = [("bytes", C.c_int64), ("device_ms", C.c_float), ("direction", C.c_int32)]


class StagedStep(C.Structure):
    _fields_ = [("slots", C.c_void_p), ("row_offsets", C.c_void_p), ("positions", C.c_void_p),
                ("page_table", C.c_void_p), ("lengths", C.c_void_p),
                ("start_positions", C.c_void_p), ("fill_pages", C.c_void_p),
                ("n_fill", C.c_int32), ("fill_seed", C.c_uint64), ("cow_pairs", C.c_void_p),
                ("n_cow", C.c_int32), ("prime_lanes", C.c_void_p), ("prime_tokens", C.c_void_p),
                ("n_prime", C.c_int32)]


_lib = None


def lib():
    """Load the HIP library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"HIP extension missing: {LIB_PATH} (run __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        P, i32, i64, u64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_float
        sig = {
            "rstr_session_open": (i32, [i32, C.POINTER(P)]),
            "rstr_session_close": (i32, [P]),
            "rstr_last_error": (C.c_char_p, [P]),
            "rstr_open_error": (C.c_char_p, []),
            "rstr_session_memory": (i32, [P, C.POINTER(i64), C.POINTER(i64)]),
            "rstr_model_bind": (i32, [P, P, P, i32, C.POINTER(P)]),
            "rstr_model_bind_synthetic": (i32, [P, P, u64, C.POINTER(P)]),
            "rstr_model_bind_raw": (i32, [P, P, P, i32, C.POINTER(P)]),
            "rstr_model_close": (i32, [P]),
            "rstr_model_weight_bytes": (i64, [P]),
            "rstr_model_export_linear": (i32, [P, i32, i32, P, P]),
            "rstr_pool_open": (i32, [P, i32, i32, C.POINTER(P)]),
            "rstr_pool_close": (i32, [P]),
            "rstr_pool_copy_page": (i32, [P, i32, i32]),
            "rstr_pool_upload": (i32, [P, i32, i32, i64, P, i64]),
            "rstr_pool_download": (i32, [P, i32, i32, i64, P, i64]),
            "rstr_pool_fill_synthetic": (i32, [P, P, i32, u64]),
            "rstr_chunk_export_submit": (i32, [P, P, i32, i32, i32, P, C.POINTER(P)]),
            "rstr_chunk_restore_submit": (i32, [P, P, i32, i32, i32, P, i32, C.POINTER(P)]),
            "rstr_transfer_done": (i32, [P]),
            "rstr_chunk_bench": (i32, [P, P, i32, i32, i32, i32, i32, C.POINTER(f32)]),
            "rstr_transfer_complete": (i32, [P, C.POINTER(TransferStats)]),
            "rstr_decoder_open": (i32, [P, P, i32, i32, i32, i32, C.POINTER(P)]),
            "rstr_decoder_close": (i32, [P]),
            "rstr_prime_lanes": (i32, [P, i32, P, P]),
            "rstr_prime_rows": (i32, [P, i32, P, P]),
            "rstr_step_lanes": (i32, [P, P, P, P, P, P, P, P]),
            "rstr_step_lanes_submit": (i32, [P, P, P, P, P, P, P]),
            "rstr_step_lanes_collect": (i32, [P, P]),
            "rstr_decode_logits": (i32, [P, P]),
            "rstr_decode_logits_device": (i32, [P, C.POINTER(P)]),
            "rstr_decoder_read_rows": (i32, [P, P]),
            "rstr_decoder_set_graph": (i32, [P, i32]),
            "rstr_decoder_step_timing": (i32, [P, P, i32]),
            "rstr_linear_run": (i32, [P, i32, i32, i32, P, P, i32, i32, P]),
            "rstr_prefill_open": (i32, [P, P, i32, i32, i32, i32, C.POINTER(P)]),
            "rstr_prefill_range": (i32, [P, P, P, P, P, i32, i32]),
            "rstr_append_run": (i32, [P, i32, i32, P, P, P]),
            "rstr_tail_run": (i32, [P, i32, i32, i32, P, P, P, P]),
            "rstr_attention_run": (i32, [P, i32, i32, i32, i32, i32, f32, P, P, P, P, i32, P, P, P]),
            "rstr_attention_run_static": (i32, [P, i32, i32, i32, i32, i32, f32, P, P, P, P, i32, P, P, P]),
            "rstr_attention_bench": (i32, [P, i32, i32, i32, i32, i32, f32, P, P, i32, P, i32,
                                           C.POINTER(f32), C.POINTER(f32)]),
            "rstr_schedule_upload": (i32, [P, P, i32]),
            "rstr_schedule_run": (i32, [P, i32, i32, P, C.POINTER(f32)]),
            "rstr_decoder_profile_steps": (i32, [P, i32, i32, P, P]),
            "rstr_kv4_open": (i32, [P, i32, i32, i32, i32, i32, C.POINTER(P)]),
            "rstr_kv4_close": (i32, [P]),
            "rstr_kv4_bytes": (i64, [P]),
            "rstr_kv4_append": (i32, [P, i32, i32, i32, P, i64, i64, P, i64, i64, P, P]),
            "rstr_kv4_read": (i32, [P, i32, i32, i32, P, P, i64, i64, P, i64, i64, P]),
            "rstr_kv4_attn_open": (i32, [P, i32, i32, i32, C.POINTER(P)]),
            "rstr_kv4_attn_close": (i32, [P]),
            "rstr_kv4_attn_run": (i32, [P, i32, i32, i32, i32, i32, i32, f32, P, i64, i64, P, P, i32, P, P, i64, i64, P]),
            "rstr_step_maps": (i32, [P, i32, i32, i32, i32, P, P, P, P, i32, P, P, P, P, P, P, P]),
            "rstr_verify_open": (i32, [P, i32, i32, i32, C.POINTER(P)]),
            "rstr_verify_close": (i32, [P]),
            "rstr_verify_run": (i32, [P, i32, i32, i32, P, i64, P, P, P, i64, P, P, P, P, P, P]),
            "rstr_pool_device": (i32, [P, i32, i32, C.POINTER(P)]),
            "rstr_pool_rope_append": (i32, [P, i32, i32, i32, P, i64, i64, P, i64, i64, i32, P, i64, i64, P, i64, i64, P, P, f32, f32, i32, P, P, P, P]),
            "rstr_pool_attn_open": (i32, [P, i32, i32, i32, C.POINTER(P)]),
            "rstr_pool_attn_close": (i32, [P]),
            "rstr_pool_attn_run": (i32, [P, i32, i32, i32, i32, i32, i32, f32, P, i64, i64, P, P, i32, P, P, i32, P, i64, i64, P]),
            "rstr_bounds_open": (i32, [P, C.POINTER(P)]),
            "rstr_bounds_close": (i32, [P]),
            "rstr_bounds_device": (i32, [P, i32, C.POINTER(P)]),
            "rstr_bounds_update": (i32, [P, i32, i32, i32, P, P, i32, P, P]),
            "rstr_select_open": (i32, [P, i32, i32, i32, i32, C.POINTER(P)]),
            "rstr_select_close": (i32, [P]),
            "rstr_select_run": (i32, [P, i32, i32, i32, i32, P, i64, i64, P, P, i32, P, i32, i32, i32, P, P]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _p(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def _i32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.int32))


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.float32))


def make_desc(cfg: dict) -> Desc:
    d = Desc()
    for name, _ in Desc._fields_:
        setattr(d, name, cfg[name])
    return d


# ---- arrays on the session's GPU ----------------------------------------------------
SESSION_STREAM = C.c_void_p(-1).value   # the session's own stream, where a stream is asked for
_ELEM = {"float32": 0, "float16": 1, "bfloat16": 2}
_codes = {}   # an array library's dtype object -> element type code, or its name


def _code(dtype):
    c = _codes.get(dtype)
    if c is None:
        name = str(dtype).replace("torch.", "")
        c = _codes[dtype] = _ELEM.get(name, name)
    return c


_lock = threading.RLock()   # views die on any thread, and inside any allocation
_late = []                  # memory whose last user has left: freed at once, or when a capture has ended


class _Stay:
    """How long a handle's memory stays: while the handle is open, while views of it live, and while memory that
    hangs on it (a pool's on its model, bounds' on their pool) stays.  ``free`` runs when the last of these has left,
    then that of what it hung on."""

    def __init__(self, free, *on):
        self.free, self.on, self.users = free, on, 1
        for x in on:
            x.join()

    def join(self):
        with _lock:
            self.users += 1

    def leave(self):
        with _lock:
            self.users -= 1
            if not self.users:
                _late.append(self)
        torch = sys.modules.get("torch")
        if _late and torch is not None and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            return  # freeing waits for the device, which would end the capture: when the next one leaves
        while True:
            with _lock:
                if not _late:
                    return
                x = _late.pop(0)
            x.free()
            for y in x.on:
                y.leave()


class DeviceView:
    """Device memory that the library owns, in the form the operators take
    (and torch's ``as_tensor``, whose tensors keep their view).  While it lives its memory does:
    closing the owner, or what that hangs on, ends the handle for calls, and the memory is
    freed once the last view of it has gone."""

    def __init__(self, ptr: int, shape, dtype: str, device: int, owner):
        self._ptr, self.shape, self.dtype, self.device, self._owner = ptr, tuple(shape), dtype, device, owner
        stay = getattr(owner, "_stay", None)
        if stay is not None:
            stay.join()
            weakref.finalize(self, stay.leave).atexit = False

    def data_ptr(self) -> int:
        return self._ptr

    def stride(self):
        out = [1]
        for n in self.shape[:0:-1]:
            out.insert(0, out[0] * n)
        return tuple(out)

    @property
    def __cuda_array_interface__(self):
        return dict(shape=self.shape, typestr="<f4" if self.dtype == "float32" else "<f2", data=(self._ptr, False), version=2)


def _device_of(x):
    """The GPU that an array lives on (its ordinal; None: not on one)."""
    d = x.device
    return d if isinstance(d, int) else d.index if getattr(d, "type", None) == "cuda" else None


def _on_device(sess, x, what):
    if _device_of(x) != sess.device:
        raise ValueError(f"{what} must be on the session's GPU ({sess.device}), got {x.device}")


# These run before every call, a dozen of them a call: one expression decides the usual case, and
# only what fails it is looked at closely.


def _flat(sess, x, what, shape, code, name):
    """The address of a contiguous device array of that element type and shape."""
    try:
        if _codes[x.dtype] == code and x.get_device() == sess.device and x.shape == shape and x.is_contiguous():
            return x.data_ptr()
    except (AttributeError, KeyError):
        pass
    _on_device(sess, x, what)
    if _code(x.dtype) != code:
        raise ValueError(f"{what} must be {name}, got {x.dtype}")
    if tuple(x.shape) != shape:
        raise ValueError(f"{what} must have the shape {shape}, got {tuple(x.shape)}")
    want = 1
    for n, st in zip(reversed(x.shape), reversed(x.stride())):
        if n > 1 and st != want:
            raise ValueError(f"{what} must be contiguous")
        want *= n
    return x.data_ptr()


def _ints(sess, x, what, shape):
    return _flat(sess, x, what, shape, "int32", "int32")


def _floats(sess, x, what, shape):
    return _flat(sess, x, what, shape, 0, "float32")


def _rows(sess, x, what, heads, hd, rows=None):
    """(address, element type, row stride, head stride) of a [rows][heads][hd] device array."""
    on = getattr(x, "get_device", None)
    if on is None or on() != sess.device:
        _on_device(sess, x, what)
    code = _codes.get(x.dtype)
    if code is None:
        code = _code(x.dtype)
    if code.__class__ is not int:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    shape = x.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != hd or (rows is not None and shape[0] != rows):
        raise ValueError(f"{what} must have the shape ({'rows' if rows is None else rows}, {heads}, {hd}), got {tuple(shape)}")
    row, head, one = x.stride()
    if one != 1:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    return x.data_ptr(), code, row, head


_raw_stream = None   # torch's current stream of a device, once torch uses the GPU


def _stream(sess, stream):
    """The raw stream of a call: what it was given (a hipStream_t address, a torch
    stream, or SESSION_STREAM), else torch's current one where torch is in use,
    else the session's own."""
    global _raw_stream
    if stream is not None:
        return getattr(stream, "cuda_stream", stream)
    if _raw_stream is None:
        torch = sys.modules.get("torch")
        if torch is None or not torch.cuda.is_initialized():
            return SESSION_STREAM
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(sess.device)


class Session:
    """A device session (raster.gpu.core/make-session)."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        rc = lib().rstr_session_open(device, C.byref(h))
        if rc != 0:
            raise RstrError(rc, lib().rstr_open_error().decode())
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_session_close, h))
        self.device = device
        self.children = []   # open models, pools, decoders (closed before the session)

    def _adopt(self, obj):
        self.children.append(obj)

    def memory(self):
        """(free, total) device bytes."""
        f, t = C.c_int64(), C.c_int64()
        self.check(lib().rstr_session_memory(self.h, C.byref(f), C.byref(t)))
        return f.value, t.value

    def check(self, rc: int):
        if rc != 0:
            raise RstrError(rc, lib().rstr_last_error(self.h).decode())

    def close(self):
        """Closes what is open on it, then itself; memory that views of it still show is freed after them."""
        if self.h:
            order = {"Decoder": 0, "Prefill": 0, "Kv4Attention": 0, "Verifier": 0, "PagedAttention": 0, "BlockSelect": 0,
                     "BlockBounds": 1, "Pool": 2, "Kv4Pool": 2, "Model": 3}
            for obj in sorted(self.children, key=lambda o: order.get(type(o).__name__, 4)):
                obj.close()
            self.children = []
            self.h = None
            self._stay.leave()

    def tail(self, logits, emb):
        """The decode tail on given logits [rows][vocab] and embedding [vocab][d]
        (decode-tail!): (tokens [rows], gathered rows [rows][d])."""
        logits, emb = _f32(logits), _f32(emb)
        rows, vocab = logits.shape
        d = emb.shape[1]
        if emb.shape[0] != vocab:
            raise ValueError("embedding rows differ from the vocabulary")
        tok = np.empty(rows, np.int32)
        out = np.empty((rows, d), np.float32)
        self.check(lib().rstr_tail_run(self.h, rows, vocab, d, _p(logits), _p(emb), _p(tok), _p(out)))
        return tok, out

    def step_maps(self, page_size: int, lengths, counts, free_pages, page_table, new_lengths, row_offsets, positions,
                  slots, taken, starts=None, stream=None):
        """The tables of a step on the GPU (rstr_step_maps): int32 device arrays; ``page_table``
        [batch][width] and everything behind it are written.  The length of ``slots``
        bounds the step's rows, that of ``free_pages`` its new pages."""
        batch, (rows,) = lengths.shape[0], slots.shape
        width, n_free = page_table.shape[1], free_pages.shape[0]
        self.check(lib().rstr_step_maps(
            self.h, page_size, batch, width, rows, _ints(self, lengths, "lengths", (batch,)),
            _ints(self, counts, "counts", (batch,)), None if starts is None else _ints(self, starts, "starts", (batch,)),
            _ints(self, free_pages, "free_pages", (n_free,)), n_free, _ints(self, page_table, "page_table", (batch, width)),
            _ints(self, new_lengths, "new_lengths", (batch,)), _ints(self, row_offsets, "row_offsets", (batch + 1,)),
            _ints(self, positions, "positions", (rows,)), _ints(self, slots, "slots", (rows,)),
            _ints(self, taken, "taken", (1,)), _stream(self, stream)))

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()


class Model:
    """Resident quantised model (decoder-gpu/bind-decode! weights)."""

    def __init__(self, sess: Session, cfg: dict, seed: int | None = None, tensors=None, raw_tensors=None):
        """``tensors``: (layer, role, f32 array); ``raw_tensors``: (layer, role,
        "F32" | "F16" | "BF16", array of the stored elements -- float32, float16
        or the bf16 bit patterns as uint16), e.g. views of a mapped checkpoint."""
        self.sess, self.cfg = sess, dict(cfg)
        self._desc = make_desc(cfg)
        h = C.c_void_p()
        if raw_tensors is not None:
            keep = []
            arr = (RawTensor * len(raw_tensors))()
            for i, (layer, role, dtype, data) in enumerate(raw_tensors):
                code = RAW_DTYPES[dtype]
                data = np.ascontiguousarray(data).reshape(-1)
                if data.itemsize != (4 if code == 0 else 2):
                    raise ValueError(f"{dtype} tensor with {data.dtype} elements")
                keep.append(data)
                arr[i] = RawTensor(layer, ROLE[role] if isinstance(role, str) else role, code,
                                   data.ctypes.data, data.size)
            rc = lib().rstr_model_bind_raw(sess.h, C.byref(self._desc), C.cast(arr, C.c_void_p),
                                           len(raw_tensors), C.byref(h))
        elif tensors is None:
            rc = lib().rstr_model_bind_synthetic(sess.h, C.byref(self._desc), int(seed), C.byref(h))
        else:
            keep = []
            arr = (Tensor * len(tensors))()
            for i, (layer, role, data) in enumerate(tensors):
                data = _f32(data).ravel()
                keep.append(data)
                arr[i] = Tensor(layer, ROLE[role] if isinstance(role, str) else role,
                                data.ctypes.data, data.size)
            rc = lib().rstr_model_bind(sess.h, C.byref(self._desc), C.cast(arr, C.c_void_p),
                                       len(tensors), C.byref(h))
        sess.check(rc)
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_model_close, h), sess._stay)
        sess._adopt(self)

    @property
    def weight_bytes(self) -> int:
        return int(lib().rstr_model_weight_bytes(self.h))

    LINEAR_FORMS = {"auto": 0, "tile": 1, "wave_gemv": 2, "wg_gemv": 3}

    def linear(self, layer: int, role: str, xq, xs, splits: int, form: str = "auto") -> np.ndarray:
        """One resident projection on int8 activations (rstr_linear_run): role
        "q" is the fused [q|k|v] tensor, "gate" the fused [gate|up] one, "embed"
        the tied head."""
        xq = np.ascontiguousarray(np.asarray(xq, np.int8))
        xs = np.ascontiguousarray(np.asarray(xs, np.float32))
        rows, k = xq.shape
        n = {"q": (self.cfg["n_q"] + 2 * self.cfg["n_kv"]) * self.cfg["head_dim"], "o": self.cfg["d_model"],
             "gate": 2 * self.cfg["d_ff"], "down": self.cfg["d_model"], "embed": self.cfg["vocab"]}[role]
        y = np.empty((rows, n), np.float32)
        self.sess.check(lib().rstr_linear_run(self.h, layer, ROLE[role], rows, _p(xq), _p(xs), splits,
                                              self.LINEAR_FORMS[form], _p(y)))
        return y

    def export_linear(self, layer: int, role: str):
        cfg = self.cfg
        from_shape = {"q": (cfg["n_q"] * cfg["head_dim"], cfg["d_model"]),
                      "k": (cfg["n_kv"] * cfg["head_dim"], cfg["d_model"]),
                      "v": (cfg["n_kv"] * cfg["head_dim"], cfg["d_model"]),
                      "o": (cfg["d_model"], cfg["n_q"] * cfg["head_dim"]),
                      "gate": (cfg["d_ff"], cfg["d_model"]), "up": (cfg["d_ff"], cfg["d_model"]),
                      "down": (cfg["d_model"], cfg["d_ff"]), "embed": (cfg["vocab"], cfg["d_model"])}
        n, k = from_shape[role]
        per = 16 if cfg["weight_bits"] == 4 else 32
        wq = np.empty((n, k // 32, per), np.uint8 if cfg["weight_bits"] == 4 else np.int8)
        ws = np.empty((n, k // 32), np.uint16)
        self.sess.check(lib().rstr_model_export_linear(self.h, layer, ROLE[role], _p(wq), _p(ws)))
        return wq, ws

    def close(self):
        """Ends the handle; the weights are freed once no pool or decoder of it is left."""
        if self.h:
            self.h = None
            _left(self)
            self._stay.leave()


class Pool:
    """fp16 page pool slabs (page-pool/open-pool! device side)."""

    def __init__(self, model: Model, page_size: int, physical_pages: int):
        self.model, self.sess = model, model.sess
        self.page_size, self.physical_pages = page_size, physical_pages
        h = C.c_void_p()
        self.sess.check(lib().rstr_pool_open(model.h, page_size, physical_pages, C.byref(h)))
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_pool_close, h), model._stay)
        self._readers = self._transfers = 0   # open plans and bounds; transfers in flight
        self.sess._adopt(self)

    @property
    def page_elems(self) -> int:
        c = self.model.cfg
        return self.page_size * c["n_kv"] * c["head_dim"]

    def copy_page(self, src: int, dst: int):
        self.sess.check(lib().rstr_pool_copy_page(self.h, src, dst))

    def upload(self, slab: int, layer: int, dst_element: int, data: np.ndarray):
        data = np.ascontiguousarray(data).view(np.uint16).ravel()
        self.sess.check(lib().rstr_pool_upload(self.h, slab, layer, dst_element, _p(data), data.size))

    def download(self, slab: int, layer: int, src_element: int = 0, elements: int | None = None):
        if elements is None:
            elements = self.physical_pages * self.page_elems - src_element
        out = np.empty(elements, np.uint16)
        self.sess.check(lib().rstr_pool_download(self.h, slab, layer, src_element, _p(out), elements))
        return out

    def pages(self, slab: int, layer: int) -> np.ndarray:
        c = self.model.cfg
        return self.download(slab, layer).view(np.float16).reshape(
            self.physical_pages, self.page_size, c["n_kv"], c["head_dim"])

    def fill_synthetic(self, pages, seed: int):
        pages = _i32(pages)
        self.sess.check(lib().rstr_pool_fill_synthetic(self.h, _p(pages), pages.size, seed))

    def append(self, layer, k_rows, v_rows, slots):
        """Routed append (paged-append run!): f32 rows -> fp16 at the given slots."""
        k_rows, v_rows, slots = _f32(k_rows), _f32(v_rows), _i32(slots)
        self.sess.check(lib().rstr_append_run(self.h, layer, slots.size, _p(k_rows), _p(v_rows),
                                              _p(slots)))

    def pages_device(self, slab: int, layer: int) -> DeviceView:
        """One slab (0: keys, 1: values) of a layer where it is, on the GPU (rstr_pool_device):
        float16 [pages][page_size][n_kv][head_dim]."""
        c, p = self.model.cfg, C.c_void_p()
        self.sess.check(lib().rstr_pool_device(self.h, slab, layer, C.byref(p)))
        return DeviceView(p.value, (self.physical_pages, self.page_size, c["n_kv"], c["head_dim"]), "float16", self.sess.device, self)

    def rope_append(self, layer: int, k, v, slots, positions=None, frequencies=None, q=None, q_out=None, q_gain=None, k_gain=None,
                    eps: float = 1e-6, gain_offset: float = 0.0, stream=None):
        """Appends device rows k, v [rows][n_kv][head_dim] to ``slots`` [rows], and writes q [rows][n_q][head_dim] to
        ``q_out`` (``q`` itself, by default), with heads of q and k normalised where a float32 gain [head_dim] is
        given and turned by ``positions`` [rows] times the float64 ``frequencies`` [rotary_dim / 2] (None: not
        turned) (rstr_pool_rope_append).  Rows whose slot is negative are not appended."""
        s, c = self.sess, self.model.cfg
        rows, hd = slots.shape[0], c["head_dim"]
        kp, kt, kr, kh = _rows(s, k, "k", c["n_kv"], hd, rows)
        vp, vt, vr, vh = _rows(s, v, "v", c["n_kv"], hd, rows)
        n_q, qs, os = 0, (None, 0, 0), (None, 0, 0)
        if q is not None:
            n_q = q.shape[1]
            qp, qt, qr, qh = _rows(s, q, "q", n_q, hd, rows)
            qs = os = qp, qr, qh
            if q_out is not None:
                op, ot, orow, oh = _rows(s, q_out, "q_out", n_q, hd, rows)
                os = op, orow, oh
                if ot != qt:
                    raise ValueError("q and q_out must have the same element type")
            if qt != kt:
                raise ValueError("q, k and v must have the same element type")
        elif q_out is not None:
            raise ValueError("q_out is given without q")
        if kt != vt:
            raise ValueError("k and v must have the same element type")
        rot, fp, pp = 0, None, None
        if frequencies is not None:
            if positions is None:
                raise ValueError("frequencies are given without positions")
            half = frequencies.shape[0]
            rot, fp = 2 * half, _flat(s, frequencies, "frequencies", (half,), "float64", "float64")
            pp = _ints(s, positions, "positions", (rows,))
        s.check(lib().rstr_pool_rope_append(
            self.h, layer, rows, kt, kp, kr, kh, vp, vr, vh, n_q, *qs, *os,
            None if q_gain is None else _floats(s, q_gain, "q_gain", (hd,)), None if k_gain is None else _floats(s, k_gain, "k_gain", (hd,)),
            eps, gain_offset, rot, fp, pp, _ints(s, slots, "slots", (rows,)), _stream(s, stream)))

    def chunk_elements(self, token_count: int) -> int:
        """Payload elements of a durable chunk of ``token_count`` tokens."""
        c = self.model.cfg
        return 2 * c["n_layers"] * token_count * c["n_kv"] * c["head_dim"]

    def export_submit(self, pages, start: int, token_count: int) -> "Transfer":
        """Gather tokens [start, start+token_count) of the route over ``pages`` into a
        durable fp16 payload (filled when the transfer completes)."""
        pages = _i32(pages).ravel()
        out = np.empty(self.chunk_elements(token_count), np.uint16)
        h = C.c_void_p()
        self.sess.check(lib().rstr_chunk_export_submit(self.h, _p(pages), pages.size, int(start), int(token_count),
                                                      _p(out), C.byref(h)))
        return Transfer(self.sess, h, out, (pages, out), self)

    def restore_submit(self, pages, start: int, token_count: int, payload) -> "Transfer":
        """Scatter a durable payload (fp16 bits as uint16, or float32) into the route's pages."""
        pages = _i32(pages).ravel()
        payload = np.ascontiguousarray(payload)
        if payload.dtype == np.float16:
            payload = payload.view(np.uint16)
        if payload.dtype == np.uint16:
            dtype = 0
        elif payload.dtype == np.float32:
            dtype = 1
        else:
            raise ValueError("Payload dtype and representation cannot be restored to FP16")
        if payload.size != self.chunk_elements(token_count):
            raise ValueError("payload length differs from its descriptor")
        h = C.c_void_p()
        self.sess.check(lib().rstr_chunk_restore_submit(self.h, _p(pages), pages.size, int(start), int(token_count),
                                                       _p(payload), dtype, C.byref(h)))
        return Transfer(self.sess, h, None, (pages, payload), self)

    def chunk_bench(self, pages, start: int, token_count: int, mode: int, iters: int) -> float:
        """Average ms of the gather (mode 0) / scatter (mode 1) kernel alone."""
        pages = _i32(pages).ravel()
        ms = C.c_float()
        self.sess.check(lib().rstr_chunk_bench(self.h, _p(pages), pages.size, int(start), int(token_count),
                                               int(mode), int(iters), C.byref(ms)))
        return ms.value

    def attention(self, layer, q, page_table, lengths, start_positions=None, positions=None,
                  window=0, scale=None, split=256, static=False):
        """Isolated routed attention (paged-attention/run!) with f32 q/out;
        ``static`` selects the allocation-free entry (rstr_attention_run_static)."""
        c = self.model.cfg
        q = _f32(q)
        B, n_q, hd = q.shape
        lengths = _i32(lengths)
        starts = _i32(start_positions if start_positions is not None else np.zeros(B))
        if positions is None:
            positions = np.where(lengths > 0, starts + lengths - 1, 0)
        pos = _i32(positions)
        pt = _i32(page_table)
        rows = _i32(np.arange(B + 1))
        out = np.empty_like(q)
        scale = c["attn_scale"] if scale is None else scale
        fn = lib().rstr_attention_run_static if static else lib().rstr_attention_run
        self.sess.check(fn(self.h, layer, B, n_q, split, window, scale, _p(q), _p(rows), _p(pos), _p(pt),
                           pt.shape[1], _p(lengths), _p(starts), _p(out)))
        return out

    def attention_bench(self, layer, q, page_table, lengths, window=0, scale=None, split=256,
                        iters=20):
        c = self.model.cfg
        q = _f32(q)
        B, n_q, hd = q.shape
        pt, lengths = _i32(page_table), _i32(lengths)
        a, b = C.c_float(), C.c_float()
        scale = c["attn_scale"] if scale is None else scale
        self.sess.check(lib().rstr_attention_bench(self.h, layer, B, n_q, split, window, scale, _p(q),
                                                   _p(pt), pt.shape[1], _p(lengths), iters,
                                                   C.byref(a), C.byref(b)))
        return a.value, b.value

    def close(self):
        """Ends the handle; refused (RstrError) while chunk transfers are in flight, or plans or bounds open.  The
        slabs are freed once no view of them, and no decoder over them, is left."""
        if self.h:
            if self._transfers:
                raise RstrError(-4, "pool has chunk transfers in flight")
            if self._readers:
                raise RstrError(-4, "pool has open attention plans or block bounds")
            self.h = None
            _left(self)
            self._stay.leave()


class Transfer:
    """A submitted chunk export/restore; keeps its host buffers alive until completion."""

    def __init__(self, sess: Session, h, payload, retained, pool: Pool):
        self.sess, self.h, self.payload, self._retained, self._pool = sess, h, payload, retained, pool
        pool._transfers += 1

    def done(self) -> bool:
        if self.h is None:  # completed
            return True
        rc = lib().rstr_transfer_done(self.h)
        if rc < 0:
            self.sess.check(rc)
        return rc == 1

    def complete(self) -> dict:
        """Wait, release the transfer; returns {bytes, device_ms, direction, payload}."""
        if self.h is None:
            raise RstrError(-4, "transfer already completed")
        st = TransferStats()
        h, self.h = self.h, None
        self._pool._transfers -= 1
        self.sess.check(lib().rstr_transfer_complete(h, C.byref(st)))
        self._retained = None
        return {"bytes": int(st.bytes), "device_ms": float(st.device_ms),
                "direction": "download" if st.direction == 1 else "upload", "payload": self.payload}


class Decoder:
    """Paged lane decoder (paged-decoder/open! + step-lanes!)."""

    def __init__(self, model: Model, pool: Pool, batch: int, pages_per_seq: int, maxpos: int,
                 split: int = 256):
        self.model, self.pool, self.sess = model, pool, model.sess
        self.batch, self.pps, self.maxpos, self.split = batch, pages_per_seq, maxpos, split
        h = C.c_void_p()
        self.sess.check(lib().rstr_decoder_open(model.h, pool.h, batch, pages_per_seq, maxpos, split,
                                                C.byref(h)))
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_decoder_close, h), pool._stay, model._stay)
        self._keep = []
        self.sess._adopt(self)

    def set_graph(self, enabled: bool):
        self.sess.check(lib().rstr_decoder_set_graph(self.h, 1 if enabled else 0))

    STEP_TIMING = ("validate", "prior_sync", "pack", "enqueue", "device_wait", "handback", "call", "device_step")

    def step_timing(self) -> dict:
        """Phases (ms) of the last step_lanes call (rstr_decoder_step_timing)."""
        out = np.zeros(len(self.STEP_TIMING), np.float64)
        self.sess.check(lib().rstr_decoder_step_timing(self.h, _p(out), out.size))
        return dict(zip(self.STEP_TIMING, out.tolist()))

    def prime_lanes(self, lanes, tokens):
        lanes, tokens = _i32(lanes), _i32(tokens)
        self.sess.check(lib().rstr_prime_lanes(self.h, lanes.size, _p(lanes), _p(tokens)))

    def prime_rows(self, lanes, rows):
        lanes, rows = _i32(lanes), _f32(rows)
        self.sess.check(lib().rstr_prime_rows(self.h, lanes.size, _p(lanes), _p(rows)))

    def step_lanes(self, slots, row_offsets, positions, page_table, lengths, start_positions):
        args = [_i32(a) for a in (slots, row_offsets, positions, page_table, lengths, start_positions)]
        out = np.empty(self.batch, np.int32)
        self.sess.check(lib().rstr_step_lanes(self.h, *[_p(a) for a in args], _p(out)))
        return out

    def step_lanes_submit(self, slots, row_offsets, positions, page_table, lengths, start_positions):
        """Enqueue one step without waiting (rstr_step_lanes_submit); at most two in flight."""
        args = [_i32(a) for a in (slots, row_offsets, positions, page_table, lengths, start_positions)]
        self.sess.check(lib().rstr_step_lanes_submit(self.h, *[_p(a) for a in args]))

    def step_lanes_collect(self) -> np.ndarray:
        """Tokens of the oldest submitted step (rstr_step_lanes_collect)."""
        out = np.empty(self.batch, np.int32)
        self.sess.check(lib().rstr_step_lanes_collect(self.h, _p(out)))
        return out

    def logits(self) -> np.ndarray:
        out = np.empty((self.batch, self.model.cfg["vocab"]), np.float32)
        self.sess.check(lib().rstr_decode_logits(self.h, _p(out)))
        return out

    def logits_device(self) -> DeviceView:
        """The last step's logits where they are, on the GPU (rstr_decode_logits_device)."""
        p = C.c_void_p()
        self.sess.check(lib().rstr_decode_logits_device(self.h, C.byref(p)))
        return DeviceView(p.value, (self.batch, self.model.cfg["vocab"]), "float32", self.sess.device, self)

    def rows(self) -> np.ndarray:
        out = np.empty((self.batch, self.model.cfg["d_model"]), np.float32)
        self.sess.check(lib().rstr_decoder_read_rows(self.h, _p(out)))
        return out

    def schedule_upload(self, steps):
        """steps: list of dicts with the six descriptors (+ optional fill_pages, fill_seed,
        cow_pairs)."""
        keep = []
        arr = (StagedStep * len(steps))()
        for i, st in enumerate(steps):
            f = {}
            for k in ("slots", "row_offsets", "positions", "page_table", "lengths", "start_positions"):
                a = _i32(st[k])
                keep.append(a)
                f[k] = a.ctypes.data
            fill = _i32(st.get("fill_pages", []))
            cow = _i32(st.get("cow_pairs", np.zeros((0, 2))))
            pl = _i32(st.get("prime_lanes", []))
            ptk = _i32(st.get("prime_tokens", []))
            keep += [fill, cow, pl, ptk]
            arr[i] = StagedStep(f["slots"], f["row_offsets"], f["positions"], f["page_table"],
                                f["lengths"], f["start_positions"],
                                fill.ctypes.data if fill.size else None, fill.size,
                                int(st.get("fill_seed", 0)),
                                cow.ctypes.data if cow.size else None, cow.size // 2,
                                pl.ctypes.data if pl.size else None,
                                ptk.ctypes.data if ptk.size else None, pl.size)
        self.sess.check(lib().rstr_schedule_upload(self.h, C.cast(arr, C.c_void_p), len(steps)))
        self._keep = keep

    def schedule_run(self, first: int, count: int):
        out = np.empty((count, self.batch), np.int32)
        ms = C.c_float()
        self.sess.check(lib().rstr_schedule_run(self.h, first, count, _p(out), C.byref(ms)))
        return out, ms.value

    def profile_steps(self, first: int, count: int):
        ms = np.zeros(len(KERNEL_CLASSES), np.float32)
        n = np.zeros(len(KERNEL_CLASSES), np.int32)
        self.sess.check(lib().rstr_decoder_profile_steps(self.h, first, count, _p(ms), _p(n)))
        return {k: (float(ms[i]), int(n[i])) for i, k in enumerate(KERNEL_CLASSES)}

    def close(self):
        """Ends the handle; its memory is freed once no view of its logits is left."""
        if self.h:
            self.h = None
            _left(self)
            self._stay.leave()


class Prefill:
    """Bulk-prefill decoder over ``rows`` tile rows (the ``:prefill-T`` link of
    paged-decoder/open!, layers only) and prefill-range!'s run."""

    def __init__(self, model: Model, pool: Pool, rows: int, pages_per_seq: int, maxpos: int,
                 split: int = 256):
        self.model, self.pool, self.sess = model, pool, model.sess
        self.rows, self.pps, self.maxpos, self.split = rows, pages_per_seq, maxpos, split
        h = C.c_void_p()
        self.sess.check(lib().rstr_prefill_open(model.h, pool.h, rows, pages_per_seq, maxpos, split,
                                                C.byref(h)))
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_decoder_close, h), pool._stay, model._stay)
        self.sess._adopt(self)

    def set_graph(self, enabled: bool):
        self.sess.check(lib().rstr_decoder_set_graph(self.h, 1 if enabled else 0))

    def prefill_range(self, tokens, slots, positions, page_table, length: int, start_position: int):
        tokens, slots, positions, page_table = (_i32(a).ravel() for a in (tokens, slots, positions, page_table))
        if tokens.size != self.rows or slots.size != self.rows or positions.size != self.rows:
            raise ValueError("Prompt tile does not match the bound prefill row count")
        if page_table.size != self.pps:
            raise ValueError("page table row does not match pages_per_seq")
        self.sess.check(lib().rstr_prefill_range(self.h, _p(tokens), _p(slots), _p(positions),
                                                 _p(page_table), int(length), int(start_position)))

    def rows_out(self) -> np.ndarray:
        """The tile's final hidden rows [rows][d_model] (before the head)."""
        out = np.empty((self.rows, self.model.cfg["d_model"]), np.float32)
        self.sess.check(lib().rstr_decoder_read_rows(self.h, _p(out)))
        return out

    def close(self):
        if self.h:
            self.h = None
            _left(self)
            self._stay.leave()


class Kv4Pool:
    """Paged K/V in 4-bit blocks (rstr_kv4_open): slots and page tables as with :class:`Pool`, at
    4.5 bits an element instead of 16."""

    def __init__(self, sess: Session, n_layers: int, n_kv: int, head_dim: int, page_size: int, physical_pages: int):
        self.sess, self.n_layers, self.n_kv, self.head_dim = sess, n_layers, n_kv, head_dim
        self.page_size, self.physical_pages = page_size, physical_pages
        h = C.c_void_p()
        sess.check(lib().rstr_kv4_open(sess.h, n_layers, n_kv, head_dim, page_size, physical_pages, C.byref(h)))
        self.h = h
        sess._adopt(self)

    @property
    def nbytes(self) -> int:
        return int(lib().rstr_kv4_bytes(self.h))

    def _kv(self, k, v, rows):
        kp, kt, kr, kh = _rows(self.sess, k, "k", self.n_kv, self.head_dim, rows)
        vp, vt, vr, vh = _rows(self.sess, v, "v", self.n_kv, self.head_dim, rows)
        if kt != vt:
            raise ValueError("k and v must have the same element type")
        return kt, (kp, kr, kh), (vp, vr, vh)

    def append(self, layer: int, k, v, slots, stream=None):
        """Quantises rows k, v [rows][n_kv][head_dim] into ``slots`` [rows] (rstr_kv4_append);
        rows whose slot is negative are skipped."""
        rows = slots.shape[0]
        t, k, v = self._kv(k, v, rows)
        self.sess.check(lib().rstr_kv4_append(self.h, layer, rows, t, *k, *v, _ints(self.sess, slots, "slots", (rows,)),
                                              _stream(self.sess, stream)))

    def read(self, layer: int, slots, k, v, stream=None):
        """Writes the values that ``slots`` hold into rows k, v (rstr_kv4_read)."""
        rows = slots.shape[0]
        t, k, v = self._kv(k, v, rows)
        self.sess.check(lib().rstr_kv4_read(self.h, layer, rows, t, _ints(self.sess, slots, "slots", (rows,)), *k, *v,
                                            _stream(self.sess, stream)))

    def close(self):
        if self.h:
            self.sess.check(lib().rstr_kv4_close(self.h))
            self.h = None
            _left(self)


class Kv4Attention:
    """Attention over a :class:`Kv4Pool` (rstr_kv4_attn_run) and its workspace: one
    call at a time, so programs and graphs that run side by side have one each."""

    def __init__(self, pool: Kv4Pool, n_q: int, max_batch: int, max_rows: int):
        self.pool, self.sess, self.n_q, self.max_batch, self.max_rows = pool, pool.sess, n_q, max_batch, max_rows
        h = C.c_void_p()
        self.sess.check(lib().rstr_kv4_attn_open(pool.h, n_q, max_batch, max_rows, C.byref(h)))
        self.h = h
        self.sess._adopt(self)

    def run(self, layer: int, q, row_offsets, page_table, lengths, out, max_rows: int | None = None, window: int = 0,
            scale: float | None = None, stream=None):
        """q, out [rows][n_q][head_dim] of one type; int32 row_offsets [batch+1], page_table
        [batch][width], lengths [batch].  ``max_rows``: the most rows of one sequence (default: all rows)."""
        s, hd = self.sess, self.pool.head_dim
        batch, rows = lengths.shape[0], q.shape[0]
        qp, t, qr, qh = _rows(s, q, "q", self.n_q, hd)
        op, ot, orow, oh = _rows(s, out, "out", self.n_q, hd, rows)
        if t != ot:
            raise ValueError("q and out must have the same element type")
        width = page_table.shape[1]
        s.check(lib().rstr_kv4_attn_run(
            self.h, layer, t, batch, rows, rows if max_rows is None else max_rows, min(window, 0x7FFFFFFF), hd ** -0.5 if scale is None else scale,
            qp, qr, qh, _ints(s, row_offsets, "row_offsets", (batch + 1,)), _ints(s, page_table, "page_table", (batch, width)),
            width, _ints(s, lengths, "lengths", (batch,)), op, orow, oh, _stream(s, stream)))

    def close(self):
        if self.h:
            self.sess.check(lib().rstr_kv4_attn_close(self.h))
            self.h = None
            _left(self)


class Verifier:
    """Verification of drafted tokens (rstr_verify_run) and its workspace: one call at a time."""

    def __init__(self, sess: Session, max_batch: int, max_rows: int, vocab: int):
        self.sess, self.max_batch, self.max_rows, self.vocab = sess, max_batch, max_rows, vocab
        h = C.c_void_p()
        sess.check(lib().rstr_verify_open(sess.h, max_batch, max_rows, vocab, C.byref(h)))
        self.h = h
        sess._adopt(self)

    def run(self, logits, row_offsets, drafts, temperature, u_accept, u_sample, accepted, tokens, draft_probs=None,
            stream=None):
        """logits [rows][vocab]; int32 row_offsets [batch+1], drafts [rows]; float32 temperature [batch],
        u_accept [rows], u_sample [batch], draft_probs [rows][vocab]; writes int32 accepted [batch] and
        tokens [rows]."""
        s = self.sess
        batch, rows = row_offsets.shape[0] - 1, drafts.shape[0]
        lp, t, lr = _matrix(s, logits, "logits", rows, self.vocab)
        pp, pr = None, 0
        if draft_probs is not None:
            pp, pt, pr = _matrix(s, draft_probs, "draft_probs", rows, self.vocab)
            if pt != 0:
                raise ValueError("draft_probs must be float32")
        s.check(lib().rstr_verify_run(
            self.h, t, batch, rows, lp, lr, _ints(s, row_offsets, "row_offsets", (batch + 1,)),
            _ints(s, drafts, "drafts", (rows,)), pp, pr, _floats(s, temperature, "temperature", (batch,)),
            _floats(s, u_accept, "u_accept", (rows,)), _floats(s, u_sample, "u_sample", (batch,)),
            _ints(s, accepted, "accepted", (batch,)), _ints(s, tokens, "tokens", (rows,)), _stream(s, stream)))

    def close(self):
        if self.h:
            self.sess.check(lib().rstr_verify_close(self.h))
            self.h = None
            _left(self)


class PagedAttention:
    """Attention over a :class:`Pool` from device arrays (rstr_pool_attn_run) and its workspace: one
    call at a time, so programs and graphs that run side by side have one each."""

    def __init__(self, pool: Pool, n_q: int, max_batch: int, max_rows: int):
        self.pool, self.sess, self.n_q, self.max_batch, self.max_rows = pool, pool.sess, n_q, max_batch, max_rows
        h = C.c_void_p()
        self.sess.check(lib().rstr_pool_attn_open(pool.h, n_q, max_batch, max_rows, C.byref(h)))
        self.h = h
        pool._readers += 1
        self.sess._adopt(self)

    def run(self, layer: int, q, row_offsets, page_table, lengths, out, max_rows: int | None = None, window: int = 0,
            scale: float | None = None, blocks=None, stream=None):
        """q, out [rows][n_q][head_dim] of one type; int32 row_offsets [batch+1], page_table
        [batch][width], lengths [batch].  ``max_rows``: the most rows of one sequence (default: all rows).
        ``blocks``: int32 [rows][n_kv][count], the blocks of the table that each row and kv head sees (None: all)."""
        s, c = self.sess, self.pool.model.cfg
        hd = c["head_dim"]
        batch, rows = lengths.shape[0], q.shape[0]
        qp, t, qr, qh = _rows(s, q, "q", self.n_q, hd)
        op, ot, orow, oh = _rows(s, out, "out", self.n_q, hd, rows)
        if t != ot:
            raise ValueError("q and out must have the same element type")
        width, bp, count = page_table.shape[1], None, 0
        if blocks is not None:
            count = blocks.shape[2]
            bp = _ints(s, blocks, "blocks", (rows, c["n_kv"], count))
        s.check(lib().rstr_pool_attn_run(
            self.h, layer, t, batch, rows, rows if max_rows is None else max_rows, min(window, 0x7FFFFFFF), hd ** -0.5 if scale is None else scale,
            qp, qr, qh, _ints(s, row_offsets, "row_offsets", (batch + 1,)), _ints(s, page_table, "page_table", (batch, width)),
            width, _ints(s, lengths, "lengths", (batch,)), bp, count, op, orow, oh, _stream(s, stream)))

    def close(self):
        if self.h:
            self.sess.check(lib().rstr_pool_attn_close(self.h))
            self.h = None
            self.pool._readers -= 1
            _left(self)


class BlockBounds:
    """The least and the greatest key element of every channel of a :class:`Pool`'s pages (rstr_bounds_open)."""

    def __init__(self, pool: Pool):
        self.pool, self.sess = pool, pool.sess
        h = C.c_void_p()
        self.sess.check(lib().rstr_bounds_open(pool.h, C.byref(h)))
        self.h = h
        self._stay = _Stay(functools.partial(lib().rstr_bounds_close, h), pool._stay)
        self._selections = 0
        pool._readers += 1
        self.sess._adopt(self)

    def update(self, layer: int, row_offsets, page_table, lengths, rows: int, stream=None):
        """Bounds of the pages in which the new rows of a step lie, ``rows`` of them at most, from the keys that are
        there (rstr_bounds_update)."""
        s, batch, width = self.sess, lengths.shape[0], page_table.shape[1]
        s.check(lib().rstr_bounds_update(
            self.h, layer, batch, rows, _ints(s, row_offsets, "row_offsets", (batch + 1,)),
            _ints(s, page_table, "page_table", (batch, width)), width, _ints(s, lengths, "lengths", (batch,)), _stream(s, stream)))

    def device(self, layer: int) -> DeviceView:
        """A layer's bounds where they are, on the GPU: float16 [pages][n_kv][2][head_dim]."""
        c, p = self.pool.model.cfg, C.c_void_p()
        self.sess.check(lib().rstr_bounds_device(self.h, layer, C.byref(p)))
        return DeviceView(p.value, (self.pool.physical_pages, c["n_kv"], 2, c["head_dim"]), "float16", self.sess.device, self)

    def close(self):
        """Ends the handle; refused (RstrError) while selections are open.  The bounds are freed once no view of them
        is left."""
        if self.h:
            if self._selections:
                raise RstrError(-4, "block bounds have open selections")
            self.h = None
            self.pool._readers -= 1
            _left(self)
            self._stay.leave()


class BlockSelect:
    """Selection of the blocks that a query reads, by the bounds of their keys (rstr_select_run), and its workspace:
    one call at a time."""

    def __init__(self, bounds: BlockBounds, n_q: int, max_batch: int, max_rows: int, max_pages: int):
        self.bounds, self.sess, self.n_q = bounds, bounds.sess, n_q
        self.max_batch, self.max_rows, self.max_pages = max_batch, max_rows, max_pages
        h = C.c_void_p()
        self.sess.check(lib().rstr_select_open(bounds.h, n_q, max_batch, max_rows, max_pages, C.byref(h)))
        self.h = h
        bounds._selections += 1
        self.sess._adopt(self)

    def run(self, layer: int, q, row_offsets, page_table, lengths, blocks, first: int = 1, last: int = 1, stream=None):
        """Writes int32 ``blocks`` [rows][n_kv][count]: for q [rows][n_q][head_dim], the blocks of highest score, the
        ``first`` first and the ``last`` last ones always among them; ascending, -1 behind the last."""
        s, c = self.sess, self.bounds.pool.model.cfg
        batch, rows, width, count = lengths.shape[0], q.shape[0], page_table.shape[1], blocks.shape[2]
        qp, t, qr, qh = _rows(s, q, "q", self.n_q, c["head_dim"])
        s.check(lib().rstr_select_run(
            self.h, layer, t, batch, rows, qp, qr, qh, _ints(s, row_offsets, "row_offsets", (batch + 1,)),
            _ints(s, page_table, "page_table", (batch, width)), width, _ints(s, lengths, "lengths", (batch,)), count, first, last,
            _ints(s, blocks, "blocks", (rows, c["n_kv"], count)), _stream(s, stream)))

    def close(self):
        if self.h:
            self.sess.check(lib().rstr_select_close(self.h))
            self.h = None
            self.bounds._selections -= 1
            _left(self)


def _matrix(sess, x, what, rows, cols):
    """(address, element type, row stride) of a [rows][cols] device array."""
    on = getattr(x, "get_device", None)
    if on is None or on() != sess.device:
        _on_device(sess, x, what)
    code = _code(x.dtype)
    if not isinstance(code, int):
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {x.dtype}")
    if tuple(x.shape) != (rows, cols):
        raise ValueError(f"{what} must have the shape ({rows}, {cols}), got {tuple(x.shape)}")
    st = x.stride()
    if cols > 1 and st[1] != 1:
        raise ValueError(f"the last dimension of {what} must be contiguous")
    return x.data_ptr(), code, st[0]


def _left(child):
    """A closed handle is no longer its session's to close."""
    if child in child.sess.children:
        child.sess.children.remove(child)
