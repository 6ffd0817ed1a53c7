"""The steps of a decoder on either side of the MoE block call, on the GPU (``include/urb_step.h``).

``AdaptedProjection``: token rows times one packed matrix (BF16, MXFP4, MXFP8) plus each row's
low-rank adapter.  ``qk_norm_rope``: the norm of every query and key head with the position
rotation.  ``Sampler``: a token per row of logits under temperature, top-k, top-p and min-p.  With
``moe.MoeLayer.forward_block`` between them, a decoder's residual stream stays on the GPU from
block to block and to the next token (attention is the caller's).

Rows are torch.bfloat16 or torch.float32 device tensors.  All compute runs in ``liburb_moe.so``; this
module only checks tensors and passes their addresses.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import numpy as np

from . import configs as C
from . import native as N
from .moe import _ptr, torch

# the urb_dtype of rows; other types are the library's to refuse
_TYPES = {} if torch is None else {torch.bfloat16: N.DTYPES["BF16"], torch.float32: N.DTYPES["F32"]}


def _type(dtype) -> int:
    return _TYPES.get(dtype, 7)


def _stream(stream, device: int) -> int:
    """The handle of a stream, or of the device's current one (the call that torch's own generated
    code makes: torch.cuda.current_stream() builds an object, 2.9 us of a 10 us call)."""
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(device)


def _bytes(t) -> int:
    return t.nbytes if isinstance(t, np.ndarray) else t.numel() * t.element_size()


def _on_host(t) -> bool:
    return isinstance(t, np.ndarray) or t.device.type == "cpu"


# the types of a matrix's values, by format, and of its scales; integers are their bits
_VALUES = {C.FMT_BF16: "bfloat16", C.FMT_MXFP4: "float4_e2m1fn_x2", C.FMT_MXFP8: "float8_e4m3fn"}
_SCALES = "float8_e8m0fnu"


def _payload(t, name: str, own: str, device: Optional[int]) -> None:
    """Refuses values of another type than ``own`` that has the same number of bytes (float16 as
    BF16, another 8-bit type) and, with ``device``, tensors that are not there."""
    if isinstance(t, np.ndarray):
        fits = t.dtype.kind in "iu" or t.dtype.name == own
    else:
        kind = t.dtype
        fits = kind == getattr(torch, own, None) or not (
            kind.is_floating_point or kind.is_complex or kind == torch.bool)
    if not fits:
        raise ValueError(f"{name} must be {own} or integers holding its bits, not {t.dtype}")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device}")


class _Current:
    """torch.cuda.device(index), entered only where another device is current."""
    __slots__ = ("index", "guard")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.guard = None
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()

    def __exit__(self, *error):
        if self.guard is not None:
            self.guard.__exit__(*error)


def _vector(t, name: str, n: int, dtype, device: int) -> Optional[int]:
    """The address of a contiguous vector of n values on the device, or None."""
    if t is None:
        return None
    if t.get_device() != device or t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on "
                         f"cuda:{device}")
    return t.data_ptr()


def _rows(t, name: str, cols: int, dtype, device: int) -> int:
    """The row stride of a [rows, cols] tensor on the device whose rows are contiguous."""
    if t.get_device() != device or t.dtype != dtype or t.dim() != 2 or t.shape[1] != cols:
        raise ValueError(f"{name} must be a {dtype} [rows, {cols}] tensor on cuda:{device}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else cols


class _Context:
    """A context of the library, on the device that is current when it is made."""
    _destroy = _sync = None

    def _make(self, create, *args) -> None:
        self.device = torch.cuda.current_device()
        ctx = ctypes.c_void_p()
        N.check(create(*args, ctypes.byref(ctx)), create.__name__)
        self._ctx = ctx

    def sync(self, stream=None) -> None:
        """Waits for the stream and raises UrbError for a failure of the calls before."""
        with _Current(self.device):
            N.check(getattr(N.moe_lib(), self._sync)(self._ctx, _stream(stream, self.device)),
                    self._sync)

    def close(self) -> None:
        if getattr(self, "_ctx", None):
            getattr(N.moe_lib(), self._destroy)(self._ctx)
            self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class AdaptedProjection(_Context):
    """y = W x + scale_a B_a (A_a x) over token rows, a = the row's adapter (``urb_proj_ctx``).

    ``data``, ``scales``: the [rows, cols] matrix in the checkpoint layout (host or device; with
    ``source`` SOURCE_DEVICE_BORROW in the panel layout of ``moe.pack_matrix``), as values of the
    format's own type or integers holding their bits.  ``dtype``: the rows' type, ``out_dtype`` the
    outputs' (the same by default).  ``slots`` adapters of up to ``max_rank`` can be held at a
    time."""

    _destroy, _sync = "urb_proj_destroy", "urb_proj_sync"

    def __init__(self, data, scales, fmt: int, rows: int, cols: int, max_tokens: int, dtype=None,
                 out_dtype=None, slots: int = 0, max_rank: int = 0, source: Optional[int] = None):
        self.rows, self.cols, self.max_tokens = rows, cols, max_tokens
        self.slots, self.max_rank = slots, max_rank
        self.dtype = torch.float32 if dtype is None else dtype
        self.out_dtype = self.dtype if out_dtype is None else out_dtype
        host = _on_host(data)
        if scales is not None and _on_host(scales) != host:
            raise ValueError("the matrix and its scales must be in the same memory")
        if source is None:
            source = N.SOURCE_HOST if host else N.SOURCE_DEVICE_COPY
        if (source == N.SOURCE_HOST) != host:
            raise ValueError("source does not match where the matrix is")
        if fmt in C.FORMAT_NAMES:
            want, want_scales = C.matrix_bytes(fmt, rows, cols)
            if _bytes(data) != want or (0 if scales is None else _bytes(scales)) != want_scales:
                raise ValueError("the matrix does not have the bytes of its format and shape")
            device = None if host else torch.cuda.current_device()
            _payload(data, "data", _VALUES[fmt], device)
            if scales is not None:
                _payload(scales, "scales", _SCALES, device)
        self._borrowed = (data, scales) if source == N.SOURCE_DEVICE_BORROW else None
        desc = N.ProjDesc(rows, cols, fmt, _type(self.dtype), _type(self.out_dtype), max_tokens,
                          slots, max_rank)
        w = N.Matrix(_ptr(data), _ptr(scales))
        self._make(N.moe_lib().urb_proj_create, ctypes.byref(desc), ctypes.byref(w), source)

    def set_adapter(self, slot: int, a, b, scale: float = 1.0, stream=None) -> None:
        """Fills a slot with a [rank, cols] and b [rows, rank] (BF16: torch.bfloat16, or 16-bit
        integers holding its bits), from host or device memory, in stream order."""
        rank = a.shape[0]
        if tuple(a.shape) != (rank, self.cols) or tuple(b.shape) != (self.rows, rank):
            raise ValueError(f"a must be [rank, {self.cols}] and b [{self.rows}, rank]")
        if _bytes(a) != 2 * rank * self.cols or _bytes(b) != 2 * rank * self.rows:
            raise ValueError("adapters are BF16")
        if _on_host(a) != _on_host(b):
            raise ValueError("a and b must be in the same memory")
        for t, name in ((a, "a"), (b, "b")):
            _payload(t, name, "bfloat16", None if _on_host(a) else self.device)
        ad = N.Adapter(_ptr(a), _ptr(b), rank, float(scale))
        source = N.SOURCE_HOST if _on_host(a) else N.SOURCE_DEVICE_COPY
        with _Current(self.device):
            N.check(N.moe_lib().urb_proj_set_adapter(self._ctx, slot, ctypes.byref(ad), source,
                                                     _stream(stream, self.device)),
                    "urb_proj_set_adapter")

    def clear_adapter(self, slot: int, stream=None) -> None:
        with _Current(self.device):
            N.check(N.moe_lib().urb_proj_set_adapter(self._ctx, slot, None, N.SOURCE_DEVICE_COPY,
                                                     _stream(stream, self.device)),
                    "urb_proj_set_adapter")

    def forward_into(self, x, y, adapter_ids=None, stream=None) -> None:
        """x [T, cols] -> y [T, rows], stream-ordered; ``adapter_ids`` [T] int32: each row's slot,
        negative for none.  Rows may be strided (parts of wider buffers)."""
        xs = _rows(x, "x", self.cols, self.dtype, self.device)
        ys = _rows(y, "y", self.rows, self.out_dtype, self.device)
        T = x.shape[0]
        if y.shape[0] != T:
            raise ValueError("x and y must have the same number of rows")
        ids = _vector(adapter_ids, "adapter_ids", T, torch.int32, self.device)
        with _Current(self.device):
            N.check(N.moe_lib().urb_proj_forward(self._ctx, x.data_ptr(), xs, ids, T, y.data_ptr(),
                                                 ys, _stream(stream, self.device)), "urb_proj_forward")

    def forward(self, x, adapter_ids=None):
        """x [T, cols] -> y [T, rows]; raises UrbError for ids that name no filled slot."""
        y = torch.empty((x.shape[0], self.rows), dtype=self.out_dtype, device=x.device)
        self.forward_into(x, y, adapter_ids)
        self.sync()
        return y

    def memory(self) -> Tuple[int, int, int]:
        """HBM bytes of the matrix (0 when borrowed), the adapter slots and the workspace."""
        n = [ctypes.c_size_t() for _ in range(3)]
        N.check(N.moe_lib().urb_proj_memory(self._ctx, *(ctypes.byref(v) for v in n)))
        return tuple(v.value for v in n)


def _heads(t, name: str, shape, dtype, device: int):
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name} must be a {dtype} {list(shape)} tensor on cuda:{device}")
    token, head, value = t.stride()
    if value != 1 and shape[2] > 1:
        raise ValueError(f"{name}: the values of a head must be contiguous")
    return token, head


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps: float,
                 zero_centered: bool = False, interleaved: bool = False, out=None, stream=None):
    """``urb_qk_norm_rope``: q [T, heads, D] and k [T, k_heads, D] (or None) normed per head by
    ``q_weight`` / ``k_weight`` [D] f32 and turned by ``positions`` [T] int64 times ``inv_freq``
    [rotary_dim / 2] f32.  Tokens and heads may be strided, as in a fused q/k/v row.  ``out``: the
    (q, k) tensors to write, which may be q and k themselves; without, new ones that belong to the
    call's stream.  Stream-ordered."""
    dtype, device, shape = q.dtype, q.get_device(), q.shape
    if q.dim() != 3 or device < 0:
        raise ValueError("q must be a [T, heads, D] tensor on a GPU")
    T, hq, D = shape
    hk = 0
    if k is not None:
        if k.dim() != 3:
            raise ValueError("k must be [T, k_heads, D]")
        hk = k.shape[1]
    k_shape = (T, hk, D)
    if out is None:   # (memory of the current stream may still be in use there)
        with torch.cuda.stream(stream):
            out = (torch.empty(shape, dtype=dtype, device=q.device),
                   None if k is None else torch.empty(k_shape, dtype=dtype, device=q.device))
    qo, ko = out
    q_in, q_out = _heads(q, "q", shape, dtype, device), _heads(qo, "q_out", shape, dtype, device)
    k_in = k_out = (0, 0)
    k_at = ko_at = kw_at = None
    if hk:
        if ko is None:
            raise ValueError("out must hold a tensor for k")
        k_in = _heads(k, "k", k_shape, dtype, device)
        k_out = _heads(ko, "k_out", k_shape, dtype, device)
        k_at, ko_at = k.data_ptr(), ko.data_ptr()
        kw_at = _vector(k_weight, "k_weight", D, torch.float32, device)
    half = 0 if inv_freq is None else inv_freq.numel()
    desc = N.QkDesc(_TYPES.get(dtype, 7), hq, hk, D, 2 * half, interleaved, zero_centered, eps,
                    *q_in, *k_in, *q_out, *k_out)
    with _Current(device):
        st = N.moe_lib().urb_qk_norm_rope(
            ctypes.byref(desc), q.data_ptr(), k_at,
            _vector(q_weight, "q_weight", D, torch.float32, device), kw_at,
            _vector(positions, "positions", T, torch.int64, device),
            _vector(inv_freq, "inv_freq", half, torch.float32, device), T, qo.data_ptr(), ko_at,
            _stream(stream, device))
    if st:
        raise N.UrbError(st, "urb_qk_norm_rope")
    return out


class Sampler(_Context):
    """Draws tokens from rows of logits over ``vocab`` tokens (``urb_sampler``)."""

    _destroy, _sync = "urb_sampler_destroy", "urb_sampler_sync"

    def __init__(self, vocab: int, max_rows: int, dtype=None):
        self.vocab, self.max_rows = vocab, max_rows
        self.dtype = torch.float32 if dtype is None else dtype
        desc = N.SamplerDesc(vocab, max_rows, _type(self.dtype))
        self._make(N.moe_lib().urb_sampler_create, ctypes.byref(desc))

    def sample_into(self, logits, uniform, ids, probs=None, temperature=None, top_k=None,
                    top_p=None, min_p=None, stream=None) -> None:
        """logits [T, vocab] (rows may be strided) and ``uniform`` [T] f32 in [0, 1) -> ``ids`` [T]
        int32 and ``probs`` [T] f32, stream-ordered.  ``temperature``, ``top_p``, ``min_p`` [T] f32
        and ``top_k`` [T] int32, each off without."""
        stride = _rows(logits, "logits", self.vocab, self.dtype, self.device)
        T, dev = logits.shape[0], self.device
        f32 = torch.float32
        params = N.SampleParams(_vector(temperature, "temperature", T, f32, dev),
                                _vector(top_k, "top_k", T, torch.int32, dev),
                                _vector(top_p, "top_p", T, f32, dev),
                                _vector(min_p, "min_p", T, f32, dev))
        with _Current(dev):
            N.check(N.moe_lib().urb_sample(
                self._ctx, logits.data_ptr(), stride, T, ctypes.byref(params),
                _vector(uniform, "uniform", T, f32, dev), _vector(ids, "ids", T, torch.int32, dev),
                _vector(probs, "probs", T, f32, dev), _stream(stream, self.device)), "urb_sample")

    def sample(self, logits, uniform, stream=None, **params):
        """-> (ids [T] int32, probs [T] f32); raises UrbError for parameters out of range.  On
        ``stream`` after what the current one holds, and waited for there."""
        ids = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
        probs = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        if stream is not None:   # the inputs and the memory of ids and probs are the current one's
            stream.wait_stream(torch.cuda.current_stream(self.device))
        self.sample_into(logits, uniform, ids, probs, stream=stream, **params)
        self.sync(stream)
        return ids, probs
