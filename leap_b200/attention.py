"""Host-side wrapper of the attention C ABI.

``AttentionContext`` owns one ``leap_ctx``: the device KV cache of a range of
layers (and of ``max_batch`` sequence slots), the RoPE table, and the split-KV
scratch.  Its methods mirror what the reference's ``run_layer`` does around
attention (src/inference/FloatTransformer.cpp:384-662) and what its
``clear_kv_cache`` does (:74-77).

Device tensors are ``torch.Tensor`` on the context's GPU (torch is used only
for device memory and streams); host arrays are ``numpy.ndarray``.  Errors
raise :class:`LeapError`, the way the reference raises std::runtime_error.
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._native import LEAP_KV_F32, LEAP_KV_Q8, CtxDesc, LeapError, check, lib

__all__ = ["AttentionContext", "LeapError", "rope_table"]


def rope_table(seq_len: int, head_dim: int, theta: float = 500000.0):
    """Reference RoPE table ``[seq_len, head_dim/2]`` (cos, sin), computed by
    the library exactly as the compiled reference does
    (src/inference/FloatTransformer.cpp:56-72)."""
    c = np.empty((seq_len, head_dim // 2), np.float32)
    s = np.empty_like(c)
    fp = ctypes.POINTER(ctypes.c_float)
    check(lib().leap_rope_table(seq_len, head_dim, ctypes.c_float(theta),
                                c.ctypes.data_as(fp), s.ctypes.data_as(fp)))
    return c, s


_torch = None  # imported with the first device tensor


def _load_torch() -> None:
    global _torch
    if _torch is None:
        import torch as _torch


def _dptr(t) -> int:
    """Device pointer of a contiguous float32 CUDA tensor."""
    _load_torch()
    torch = _torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("expected a CUDA torch.Tensor")
    if t.dtype != torch.float32 or not t.is_contiguous():
        raise TypeError("expected a contiguous float32 tensor")
    return t.data_ptr()


KV_KINDS = {"f32": LEAP_KV_F32, "q8": LEAP_KV_Q8}


def kv_kind(kv: str) -> int:
    if kv not in KV_KINDS:
        raise ValueError(f"kv must be one of {sorted(KV_KINDS)}, got {kv!r}")
    return KV_KINDS[kv]


def _ints(a, name: str, n: int | None = None) -> np.ndarray:
    """A 1-D host int32 array (kept as it is when it is one already) of whole
    numbers, none of which the conversion may change."""
    if isinstance(a, list) and all(type(x) is int and -2**31 <= x < 2**31 for x in a):
        a = np.array(a, np.int32)
    elif not isinstance(a, np.ndarray) or a.dtype != np.int32:
        wide = np.asarray(a)
        if wide.size and wide.dtype.kind not in "iu":
            raise ValueError(f"{name} must be whole numbers of 32 bits")
        a = wide.astype(np.int32)
        if (a != wide).any():
            raise ValueError(f"{name} must be whole numbers of 32 bits")
    a = np.ascontiguousarray(a)
    if a.ndim != 1 or (n is not None and a.shape[0] != n):
        raise ValueError(f"{name} must be 1-D" + ("" if n is None else f" of length {n}"))
    return a


def _iptr(a: np.ndarray) -> int:
    """Address of a contiguous host array (cheaper than ``a.ctypes.data``)."""
    return a.__array_interface__["data"][0]


def _total(a: np.ndarray) -> int:
    """Sum of the lengths (negative ones, which the library refuses, as 0)."""
    t = a.tolist()
    return sum(t) if not t or min(t) >= 0 else sum(x for x in t if x > 0)


def _hptr(a: np.ndarray) -> int:
    if a.dtype != np.float32 or not a.flags["C_CONTIGUOUS"]:
        raise TypeError("expected a C-contiguous float32 array")
    return a.ctypes.data


class AttentionContext:
    """Device attention state for ``n_layers`` layers and ``max_batch`` slots.

    Parameters follow the reference ``Config`` (src/inference/Config.h):
    ``n_heads``, ``n_kv_heads``, ``head_dim`` (= dim / n_heads), ``max_seq``
    (= seq_len).  ``rope_cos``/``rope_sin`` default to :func:`rope_table`
    with ``theta``.

    ``kv`` says how cached rows are kept: ``"f32"``, or ``"q8"`` for 8-bit
    codes with one scale for each row and kv head (``leap_ctx_create_kv``).
    Every method works on both; :meth:`decode_tree` on ``"q8"`` only.
    """

    def __init__(self, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 max_seq: int, max_batch: int = 1, device: int = 0, layer0: int = 0,
                 theta: float = 500000.0, rope_cos=None, rope_sin=None,
                 bind_torch_stream: bool = True, kv: str = "f32"):
        kind = kv_kind(kv)
        if rope_cos is None or rope_sin is None:
            rope_cos, rope_sin = rope_table(max_seq, head_dim, theta)
        self.rope_cos = np.ascontiguousarray(rope_cos, np.float32)
        self.rope_sin = np.ascontiguousarray(rope_sin, np.float32)
        if self.rope_cos.shape != (max_seq, head_dim // 2):
            raise ValueError("rope tables must be [max_seq, head_dim/2]")
        fp = ctypes.POINTER(ctypes.c_float)
        desc = CtxDesc(n_layers, layer0, n_heads, n_kv_heads, head_dim, max_seq,
                       max_batch, device, self.rope_cos.ctypes.data_as(fp),
                       self.rope_sin.ctypes.data_as(fp))
        h = ctypes.c_void_p()
        check(lib().leap_ctx_create_kv(ctypes.byref(desc), kind, ctypes.byref(h)))
        self._h = h
        self.n_layers, self.n_heads, self.n_kv_heads = n_layers, n_heads, n_kv_heads
        self.head_dim, self.max_seq, self.max_batch = head_dim, max_seq, max_batch
        self.device = device
        self.kv = kv
        self._stream = self._raw = None  # the torch stream bound, if any, and its handle
        if bind_torch_stream:
            self.bind_torch_stream()

    # -- lifetime ---------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_h", None):
            check(lib().leap_ctx_destroy(self._h))
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> ctypes.c_void_p:
        if not self._h:
            raise LeapError(1, "context is closed")
        return self._h

    # -- streams ----------------------------------------------------------
    def bind_torch_stream(self, stream=None) -> None:
        """Order this context's work on a torch CUDA stream (default: the
        current stream of its device), so torch tensors can be passed
        without extra synchronisation.  Tensors that methods return belong to
        that stream, whichever is current."""
        import torch
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        check(lib().leap_ctx_set_stream(self.handle, ctypes.c_void_p(stream.cuda_stream)))
        self._stream, self._raw = stream, stream.cuda_stream

    def use_own_stream(self) -> None:
        check(lib().leap_ctx_use_own_stream(self.handle))
        self._stream = self._raw = None

    def _foreign(self) -> bool:
        """Whether another stream than the bound one is current.  What methods
        return is allocated on the stream that writes it: another stream's
        allocator may hand out memory that work still queued there reads."""
        return self._raw is not None and self._raw != _torch._C._cuda_getCurrentRawStream(self.device)

    def _like(self, q):
        _load_torch()
        if self._foreign():
            with _torch.cuda.stream(self._stream):
                return _torch.empty_like(q)
        return _torch.empty_like(q)

    def sync(self) -> None:
        check(lib().leap_sync(self.handle))

    def device_bytes(self) -> int:
        n = ctypes.c_size_t()
        check(lib().leap_ctx_device_bytes(self.handle, ctypes.byref(n)))
        return n.value

    # -- cache ------------------------------------------------------------
    def clear_kv_cache(self) -> None:
        """FloatTransformer::clear_kv_cache (FloatTransformer.cpp:74-77)."""
        check(lib().leap_kv_clear(self.handle))

    def kv_write(self, slot: int, layer: int, pos0: int, k, v) -> None:
        """Write rows [pos0, pos0+n) from reference layout [n, n_kv, hd]."""
        if isinstance(k, np.ndarray):
            k = np.ascontiguousarray(k, np.float32)
            v = np.ascontiguousarray(v, np.float32)
            n = k.shape[0]
            check(lib().leap_kv_write(self.handle, slot, layer, pos0, n, _hptr(k),
                                      _hptr(v), 1))
        else:
            n = k.shape[0]
            check(lib().leap_kv_write(self.handle, slot, layer, pos0, n, _dptr(k),
                                      _dptr(v), 0))

    def kv_read(self, slot: int, layer: int, pos0: int, n: int):
        """Rows [pos0, pos0+n) as host arrays [n, n_kv, hd] (K, V)."""
        k = np.empty((n, self.n_kv_heads, self.head_dim), np.float32)
        v = np.empty_like(k)
        check(lib().leap_kv_read(self.handle, slot, layer, pos0, n, _hptr(k), _hptr(v), 1))
        return k, v

    def kv_read_device(self, slot: int, layer: int, pos0: int, n: int):
        """The same as device tensors, on the context's stream."""
        k, v = self._rows(n)
        check(lib().leap_kv_read(self.handle, slot, layer, pos0, n, k.data_ptr(), v.data_ptr(), 0))
        return k, v

    def kv_read_packed(self, layer: int, slots, pos0, n_tok):
        """Rows [pos0[i], pos0[i]+n_tok[i]) of slots[i], one sequence after
        another, as device tensors [sum n_tok, n_kv, hd] (K, V): one launch."""
        slots = _ints(slots, "slots")
        n = slots.shape[0]
        pos0, n_tok = _ints(pos0, "pos0", n), _ints(n_tok, "n_tok", n)
        k, v = self._rows(_total(n_tok))
        check(lib().leap_kv_read_packed(self.handle, layer, n, _iptr(slots),
                                        _iptr(pos0), _iptr(n_tok), k.data_ptr(),
                                        v.data_ptr()))
        return k, v

    def kv_keep(self, slots, positions, n_keep, nodes) -> None:
        """Keep rows positions[i] + nodes (strictly increasing, n_keep[i] of
        them for each sequence) as rows positions[i], positions[i]+1, ... in
        every layer: the accepted path after :meth:`decode_tree`."""
        slots = _ints(slots, "slots")
        n = slots.shape[0]
        positions, n_keep = _ints(positions, "positions", n), _ints(n_keep, "n_keep", n)
        nodes = _ints(nodes, "nodes", _total(n_keep))
        check(lib().leap_kv_keep(self.handle, n, _iptr(slots), _iptr(positions),
                                 _iptr(n_keep), _iptr(nodes)))

    def _rows(self, n: int):
        _load_torch()
        shape, dev = (max(n, 0), self.n_kv_heads, self.head_dim), _torch.device("cuda", self.device)
        if self._raw is None:  # torch cannot order its memory on the context's own stream
            _torch.cuda.current_stream(dev).synchronize()
        elif self._foreign():
            with _torch.cuda.stream(self._stream):
                return (_torch.empty(shape, dtype=_torch.float32, device=dev),
                        _torch.empty(shape, dtype=_torch.float32, device=dev))
        return (_torch.empty(shape, dtype=_torch.float32, device=dev),
                _torch.empty(shape, dtype=_torch.float32, device=dev))

    # -- attention ----------------------------------------------------------
    def decode(self, layer: int, pos: int, q, k_new, v_new, out=None):
        """Fused RoPE + append + attention for one token (device tensors)."""
        if out is None:
            out = self._like(q)
        check(lib().leap_attn_decode(self.handle, layer, pos, _dptr(q), _dptr(k_new),
                                     _dptr(v_new), _dptr(out)))
        return out

    def decode_host(self, layer: int, pos: int, q: np.ndarray, k_new: np.ndarray,
                    v_new: np.ndarray) -> np.ndarray:
        """Same as :meth:`decode` on host arrays; blocks until done."""
        q = np.ascontiguousarray(q, np.float32)
        k_new = np.ascontiguousarray(k_new, np.float32)
        v_new = np.ascontiguousarray(v_new, np.float32)
        out = np.empty((self.n_heads, self.head_dim), np.float32)
        check(lib().leap_attn_decode_host(self.handle, layer, pos, _hptr(q), _hptr(k_new),
                                          _hptr(v_new), _hptr(out)))
        return out

    def decode_batched(self, layer: int, slots, positions, q, k_new, v_new, out=None):
        """Ragged batch: token i of slot slots[i] at positions[i]."""
        slots = np.ascontiguousarray(slots, np.int32)
        positions = np.ascontiguousarray(positions, np.int32)
        if slots.shape != positions.shape or slots.ndim != 1:
            raise ValueError("slots and positions must be equal-length 1-D")
        if out is None:
            out = self._like(q)
        check(lib().leap_attn_decode_batched(
            self.handle, layer, slots.shape[0], _iptr(slots), _iptr(positions), _dptr(q),
            _dptr(k_new), _dptr(v_new), _dptr(out)))
        return out

    def prefill(self, slot: int, layer: int, pos0: int, q, k, v, out=None):
        """Causal prefill of q.shape[0] tokens starting at pos0."""
        if out is None:
            out = self._like(q)
        check(lib().leap_attn_prefill(self.handle, slot, layer, pos0, int(q.shape[0]),
                                      _dptr(q), _dptr(k), _dptr(v), _dptr(out)))
        return out

    def _packed(self, total: int, q, k, v, out):
        """Device pointers of a ragged call's tensors, their shapes checked."""
        qs, ks = (total, self.n_heads, self.head_dim), (total, self.n_kv_heads, self.head_dim)
        ptrs = [_dptr(q), _dptr(k), _dptr(v)]
        if out is None:
            out = self._like(q)
        ptrs.append(_dptr(out))
        for name, t, shape in (("q", q, qs), ("k", k, ks), ("v", v, ks), ("out", out, qs)):
            if t.shape != shape:
                raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
            if t.get_device() != self.device:
                raise ValueError(f"{name} must be on cuda:{self.device}, got {t.device}")
        return (*ptrs, out)

    def prefill_packed(self, layer: int, slots, pos0, n_tok, q, k, v, out=None):
        """Causal prefill of several prompts (or parts of prompts): sequence i
        brings n_tok[i] tokens for slots[i] behind pos0[i] cached rows; q, k, v
        hold the sequences' tokens one after another."""
        slots = _ints(slots, "slots")
        n = slots.shape[0]
        pos0, n_tok = _ints(pos0, "pos0", n), _ints(n_tok, "n_tok", n)
        qp, kp, vp, op, out = self._packed(_total(n_tok), q, k, v, out)
        check(lib().leap_attn_prefill_packed(self.handle, layer, n, _iptr(slots),
                                             _iptr(pos0), _iptr(n_tok), qp, kp, vp, op))
        return out

    def decode_tree(self, layer: int, slots, positions, n_nodes, parents, q, k, v, out=None):
        """Attention of drafted token trees: sequence i brings n_nodes[i] nodes
        behind positions[i] cached rows.  ``parents`` holds each node's parent
        within its sequence (-1: none; parents come before children), all
        sequences' nodes one after another.  A node sees the cached rows, its
        ancestors and itself; its k and v are appended as row positions[i] +
        node.  ``kv="q8"`` only."""
        slots = _ints(slots, "slots")
        n = slots.shape[0]
        positions, n_nodes = _ints(positions, "positions", n), _ints(n_nodes, "n_nodes", n)
        total = _total(n_nodes)
        parents = _ints(parents, "parents", total)
        qp, kp, vp, op, out = self._packed(total, q, k, v, out)
        check(lib().leap_attn_tree(self.handle, layer, n, _iptr(slots), _iptr(positions),
                                   _iptr(n_nodes), _iptr(parents), qp, kp, vp, op))
        return out

    def set_decode_impl(self, impl: int) -> None:
        """0 = auto, 1 = split-KV, 2 = cluster kernel, 3 = wide split-KV,
        4 = split-KV with a separate combine launch."""
        check(lib().leap_set_decode_impl(self.handle, impl))

    def cluster_capacity(self) -> int:
        n = ctypes.c_int()
        check(lib().leap_decode_cluster_capacity(self.handle, ctypes.byref(n)))
        return n.value

    def set_overlap(self, enable: bool) -> None:
        """Let a decode launch stream its K/V while the previous kernel
        finishes (programmatic dependent launch); on by default."""
        check(lib().leap_set_overlap(self.handle, int(bool(enable))))

    def set_prefill_impl(self, impl: int) -> None:
        """0 = tensor-core 3xTF32 kernel pipelined across warp roles,
        1 = CUDA-core FP32 kernel, 2 = tensor-core 3xTF32 kernel, one tile at
        a time, 3 = the pipelined kernel with its two correction products in
        BF16 (the default)."""
        check(lib().leap_set_prefill_impl(self.handle, impl))
