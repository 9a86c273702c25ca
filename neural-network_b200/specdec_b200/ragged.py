"""Operators of a ragged decode step over an 8-bit paged cache: ``KV8.plan``
(block tables and slot maps), ``KV8.append`` and ``KV8.gather`` (cache rows),
``KV8.attend`` and ``sample``.  include/specdec.h has their definitions.

Buffers are CUDA tensors: any object with ``data_ptr()``, ``shape``,
``stride()``, ``dtype``, ``is_cuda``, ``get_device()`` and ``is_contiguous()``,
as torch's are, on the device of the cache (``sample``: of the logits).
``stream`` is a raw cudaStream_t (0: the device's default stream, torch's
current one unless a caller changed it); tensors must be ready on it.
Failures raise ``SpecDecError`` (a RuntimeError), wrong arguments before the
call ``ValueError``.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import specdec_b200 as _sd

_ROWS = {"float32": _sd.F32, "bfloat16": _sd.BF16}
_names: dict = {}  # dtype object -> its name


def _name_of(dtype) -> str:
    name = _names.get(dtype)
    if name is None:
        name = _names[dtype] = str(dtype).rpartition(".")[2]
    return name


def _dtype_of(t) -> int:
    d = _ROWS.get(_name_of(t.dtype))
    if d is None:
        raise ValueError(f"rows must be float32 or bfloat16, not {t.dtype}")
    return d


def _buffer(t, name: str, dtype: str, shape=None, device=None):
    """The address of a contiguous buffer of the given type (and shape and device)."""
    if (_names.get(t.dtype) or _name_of(t.dtype)) != dtype or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{name} must be a contiguous {dtype} CUDA tensor")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} must be a tensor of CUDA device {device}")
    return t.data_ptr()


def _optional(t, name: str, dtype: str, shape=None, device=None):
    return None if t is None else _buffer(t, name, dtype, shape, device)


def _one_device(tensors) -> int:
    devices = {t.get_device() for t in tensors if t is not None}
    if len(devices) != 1:
        raise ValueError("the tensors must be on one device")
    return devices.pop()


class KV8Layer:
    """One layer's cache: codes k, v [pages][kv heads][page tokens][head dim]
    int8 and scales [pages][kv heads][blocks of a page] float32."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k_scale.dim() != 3:
            raise ValueError("codes have 4 dimensions, scales 3")
        if tuple(k_scale.shape[:2]) != tuple(k.shape[:2]):
            raise ValueError("scales and codes must agree on pages and kv heads")
        self.shape, self.blocks = tuple(k.shape), k_scale.shape[2]
        self.record = _sd._KV8Layer(_buffer(k, "k", "int8"), _buffer(v, "v", "int8", k.shape),
                                    _buffer(k_scale, "k_scale", "float32"),
                                    _buffer(v_scale, "v_scale", "float32", k_scale.shape), k.shape[0])
        self.ptr = C.addressof(self.record)
        self._keep = (k, v, k_scale, v_scale)
        self.device = _one_device(self._keep)


class KV8Batch:
    """The requests of a step: table [requests][columns], kv_len [requests],
    cu_q [requests + 1] (int32), and for ``KV8.plan`` tok_req, tok_pos (int32),
    slots (int64) of one length and status [1] (int32)."""

    def __init__(self, table, kv_len, cu_q, tok_req=None, tok_pos=None, slots=None, status=None):
        if table.dim() != 2:
            raise ValueError("table has 2 dimensions")
        n = table.shape[0]
        rows = 0 if slots is None else slots.shape[0]
        self.n_requests = n
        self.planned = status is not None
        self.record = _sd._KV8Batch(
            _buffer(table, "table", "int32"), n, table.shape[1], _buffer(kv_len, "kv_len", "int32", (n,)),
            _buffer(cu_q, "cu_q", "int32", (n + 1,)), _optional(tok_req, "tok_req", "int32", (rows,)),
            _optional(tok_pos, "tok_pos", "int32", (rows,)), _optional(slots, "slots", "int64"), rows,
            _optional(status, "status", "int32", (1,)))
        self.ptr = C.addressof(self.record)
        self._keep = (table, kv_len, cu_q, tok_req, tok_pos, slots, status)
        self.device = _one_device(self._keep)


def _rows(t, heads: int, dim: int, name: str, device: int):
    """(address, row stride, head stride) of rows [n][heads][dim] with adjacent dims."""
    sh, st = t.shape, t.stride()
    if t.get_device() != device:
        raise ValueError(f"{name} must be a tensor of CUDA device {device}")
    if len(sh) != 3 or sh[1] != heads or sh[2] != dim or st[2] != 1:
        raise ValueError(f"{name} must be rows of {heads} heads x {dim} adjacent values, not {tuple(sh)}")
    return t.data_ptr(), st[0], st[1]


class KV8:
    """Geometry and workspace of an 8-bit paged cache with a scale per
    block_tokens positions and kv head, on one device."""

    def __init__(self, n_heads: int, n_kv_heads: int, head_dim: int, page_tokens: int = 128, block_tokens: int = 16,
                 max_batch: int = 256, device: int = 0):
        lib = _sd.load_library()
        cfg = _sd._KV8Config(n_heads, n_kv_heads, head_dim, page_tokens, block_tokens, max_batch)
        h = C.c_void_p()
        rc = lib.specdec_kv8_create(C.byref(cfg), device, C.byref(h))
        if rc:
            raise _sd.SpecDecError(rc, lib.specdec_kv8_last_error(None).decode())
        self._lib, self.h, self.device = lib, h, device
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.page_tokens, self.block_tokens = page_tokens, block_tokens

    def close(self):
        if getattr(self, "h", None):
            self._lib.specdec_kv8_destroy(self.h)
            self.h = None

    def __del__(self):
        self.close()

    def _check(self, rc: int):
        if rc:
            raise _sd.SpecDecError(rc, self._lib.specdec_kv8_last_error(self.h).decode())

    def _layer(self, layer: KV8Layer) -> int:
        if layer.shape[1:] != (self.n_kv_heads, self.page_tokens, self.head_dim) or \
                layer.blocks * self.block_tokens != self.page_tokens:
            raise ValueError(f"the layer's codes {layer.shape} and {layer.blocks} blocks a page do not fit this handle")
        if layer.device != self.device:
            raise ValueError(f"the layer must be on CUDA device {self.device}")
        return layer.ptr

    def _batch(self, batch: KV8Batch) -> int:
        if batch.device != self.device:
            raise ValueError(f"the batch must be on CUDA device {self.device}")
        return batch.ptr

    def plan(self, batch: KV8Batch, held, keep, q_len, ring, ring_state, ring_state_out, stream: int = 0) -> None:
        """Pages, lengths, row and slot maps of a step (specdec_kv8_plan)."""
        n, d = (batch.n_requests,), self.device
        self._check(self._lib.specdec_kv8_plan(
            self.h, self._batch(batch), _buffer(held, "held", "int32", n, d), _buffer(keep, "keep", "int32", n, d),
            _buffer(q_len, "q_len", "int32", n, d), _buffer(ring, "ring", "int32", None, d), ring.shape[0],
            _buffer(ring_state, "ring_state", "int32", (2,), d),
            _buffer(ring_state_out, "ring_state_out", "int32", (2,), d), stream or None))

    def append(self, layer: KV8Layer, batch: KV8Batch, k, v, stream: int = 0) -> None:
        """Writes rows k, v [rows][kv heads][head dim] to the requests' last positions."""
        kp, kr, kh = _rows(k, self.n_kv_heads, self.head_dim, "k", self.device)
        vp, vr, vh = _rows(v, self.n_kv_heads, self.head_dim, "v", self.device)
        if v.shape[0] != k.shape[0] or v.dtype != k.dtype:
            raise ValueError("k and v must have the same rows and type")
        self._check(self._lib.specdec_kv8_append(self.h, self._layer(layer), self._batch(batch), kp, kr, kh, vp, vr, vh,
                                                 _dtype_of(k), k.shape[0], stream or None))

    def gather(self, layer: KV8Layer, rows, out_k=None, out_v=None, stream: int = 0) -> None:
        """Values of the cache slots `rows` (int64) into out_k, out_v [rows][kv heads][head dim]."""
        n = rows.shape[0]
        shape = (n, self.n_kv_heads, self.head_dim)
        outs = [t for t in (out_k, out_v) if t is not None]
        if not outs:
            return
        if any(t.shape != shape or not t.is_contiguous() or t.dtype != outs[0].dtype or t.get_device() != self.device
               for t in outs):
            raise ValueError(f"outputs must be contiguous, on CUDA device {self.device}, of one type and shape {shape}")
        self._check(self._lib.specdec_kv8_gather(
            self.h, self._layer(layer), _buffer(rows, "rows", "int64", None, self.device), n, None if out_k is None else out_k.data_ptr(),
            None if out_v is None else out_v.data_ptr(), _dtype_of(outs[0]), stream or None))

    def attend(self, layer: KV8Layer, batch: KV8Batch, q, out, lse=None, max_q: Optional[int] = None,
               scale: Optional[float] = None, window: int = 0, stream: int = 0) -> None:
        """Attention of q [rows][heads][head dim] over the cache into out (and lse
        [rows][heads] float32); scale defaults to 1 / sqrt(head dim).  max_q,
        the most rows of one request, chooses the kernel: by default the mean,
        right for a batch of equal requests and for one prompt."""
        qp, qr, qh = _rows(q, self.n_heads, self.head_dim, "q", self.device)
        op, orow, oh = _rows(out, self.n_heads, self.head_dim, "out", self.device)
        if out.shape[0] != q.shape[0] or out.dtype != q.dtype:
            raise ValueError("q and out must have the same rows and type")
        lp = None if lse is None else _buffer(lse, "lse", "float32", q.shape[:2], self.device)
        if max_q is None:
            max_q = -(-q.shape[0] // max(1, batch.n_requests))
        self._check(self._lib.specdec_kv8_attend(
            self.h, self._layer(layer), self._batch(batch), qp, qr, qh, _dtype_of(q), q.shape[0], op, orow, oh, lp,
            max_q, 1.0 / math.sqrt(self.head_dim) if scale is None else scale, window, stream or None))

    def check(self, stream: int = 0) -> None:
        """Waits for the stream; raises if a wait inside an attend call on it gave up."""
        self._check(self._lib.specdec_kv8_check(self.h, stream or None))


def sample(logits, u, tokens, probs=None, temperature=None, top_k=None, top_p=None, min_p=None,
           stream: int = 0) -> None:
    """One token per row of logits [rows][vocab] from the uniforms u (specdec_sample):
    tokens int32, probs float32 [rows]; the parameters are [rows] tensors or None."""
    sh, st = logits.shape, logits.stride()
    if len(sh) != 2 or (st[1] != 1 and sh[1] > 1) or not logits.is_cuda:
        raise ValueError("logits must be rows of adjacent values on a CUDA device")
    n, d = (sh[0],), logits.get_device()
    lib = _sd.load_library()
    rc = lib.specdec_sample(
        logits.data_ptr(), _dtype_of(logits), sh[0], sh[1], st[0],
        _optional(temperature, "temperature", "float32", n, d), _optional(top_k, "top_k", "int32", n, d),
        _optional(top_p, "top_p", "float32", n, d), _optional(min_p, "min_p", "float32", n, d),
        _buffer(u, "u", "float32", n, d), _buffer(tokens, "tokens", "int32", n, d),
        _optional(probs, "probs", "float32", n, d), stream or None)
    if rc:
        raise _sd.SpecDecError(rc, lib.specdec_last_error(None).decode())
