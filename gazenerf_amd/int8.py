"""8-bit rows: a cache of feature maps and the linear layers / 1x1 convolutions that read it, for inference.

A *row* is the channel vector of one pixel (or one token): signed bytes and one fp32 scale (include/gnr.h):

    a = max(max_k |x_k|, 2^-100)     scale = a / 127     q_k = rint(x_k * (127 / a))     in fp32, ties to even

A viewer or a sweep shows the same views again and again, and rendering a view's feature map costs some twenty times as much as
turning it into an image.  ``FeatureMapCache`` keeps maps in the form the next product reads (258 channels: 276 bytes a pixel
instead of 1032), ``int8_linear`` multiplies them -- or floating maps / rows, which it quantises on the way -- with 8-bit weights
(one scale a channel, ``quantize_rows`` of the weight matrix) on the integer matrix units, and ``NeuralRendererAMD(...,
precision="int8")`` runs its 1x1 convolutions that way.

    write_featmaps(q, scale, slots, maps)            maps [B, C, P] -> slots of a cache
    read_featmaps(q, scale, slots)                   slots -> maps [B, C, P]
    quantize_rows(x)                                 [..., K] or [B, K, ...] -> QuantizedRows(q, scale)
    int8_linear(x, w_q, w_scale, bias, ...)          rows, maps or cached rows -> act(x w^T + bias)

Floating tensors are float32, bfloat16 or float16.  CUDA (ROCm) tensors only; the work goes to the current stream of their
device.  There is no backward: a call on inputs that would need a gradient, of either mode, is refused, and so is a call under
``torch.jit.trace``, which would record its result as a constant.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib, _torch_ext
from .render import _ext_call, _has_tangent, _stream_ptr

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int8: 3}
ROW_ALIGN = 16           # rows that a product reads stand on multiples of 16 bytes (a cache: 275 bytes of 258 channels and a scale on 272 + 4)
LINE = 64                # rows that this module makes for a product: a step of K never crosses a line (28672 x 516 -> 1032: 41 -> 38 us)


class QuantizedRows(NamedTuple):
    """q int8 [..., K] on a pitch of 64 bytes, scale float32 [...]."""
    q: torch.Tensor
    scale: torch.Tensor


def row_pitch(channels: int, align: int = LINE) -> int:
    """Bytes from one row to the next: a multiple of 64 in what this module makes for a product, of 16 in a cache."""
    return -(-int(channels) // align) * align


def empty_rows(*shape, device) -> torch.Tensor:
    """Uninitialised int8 rows ``shape`` = (..., K) on their pitch."""
    return torch.empty(*shape[:-1], row_pitch(shape[-1]), dtype=torch.int8, device=device)[..., :shape[-1]]


# ---- checks (the C++ binding has its own; these name the argument) -------------------------------------------------------------
def _tensor(name, t, dtypes, dims=None):
    if not torch.is_tensor(t):
        raise TypeError("%s must be a tensor" % name)
    if t.dtype not in dtypes:
        raise TypeError("%s must be %s, got %s" % (name, " / ".join(str(d)[6:] for d in dtypes), t.dtype))
    if dims is not None and t.dim() not in dims:
        raise ValueError("%s must have %s dimensions, got shape %s" % (name, " or ".join(map(str, dims)), tuple(t.shape)))


def _one_device(**ts):
    ts = {k: t for k, t in ts.items() if t is not None}
    for k, t in ts.items():
        if not t.is_cuda:
            raise RuntimeError("%s must live on a CUDA/ROCm device (the 8-bit operators have no CPU path)" % k)
    if len({t.device for t in ts.values()}) > 1:
        raise RuntimeError("all tensors must live on one device, got %s" % {k: str(t.device) for k, t in ts.items()})


def _no_grad(what, *ts):
    # a call of one row takes 5 us: torch.jit.is_tracing() at a third of its time, and no look at the tensors while no dual level is open
    if torch._C._is_tracing():
        raise RuntimeError("%s cannot be traced: the trace would hold its result as a constant" % what)
    if forward_ad._current_level >= 0 and _has_tangent(*ts):
        raise RuntimeError("%s has no forward-mode gradient: call it on inputs without a tangent (torch.autograd.forward_ad)" % what)
    if torch.is_grad_enabled():
        for t in ts:
            if getattr(t, "requires_grad", False):
                raise RuntimeError("%s has no backward: call it under torch.no_grad() or on detached tensors" % what)


_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check_cache(q, scale, slots, maps_shape):
    _tensor("q", q, (torch.int8,), (3,))
    _tensor("scale", scale, (torch.float32,), (2,))
    _tensor("slots", slots, (torch.int64,), (1,))
    n, p, c = q.shape
    if n < 1 or p < 1 or c < 1:
        raise ValueError("the cache is empty: q %s" % (tuple(q.shape),))
    if tuple(scale.shape) != (n, p):
        raise ValueError("scale must have shape %s, got %s" % ((n, p), tuple(scale.shape)))
    if (c > 1 and q.stride(2) != 1) or (p > 1 and q.stride(1) < c) or (n > 1 and q.stride(0) < (p - 1) * q.stride(1) + c):
        raise ValueError("q must have its channels contiguous and its rows apart, got strides %s" % (q.stride(),))
    if (p > 1 and scale.stride(1) != 1) or (n > 1 and scale.stride(0) < p):
        raise ValueError("scale must have its pixels contiguous and its slots apart, got strides %s" % (scale.stride(),))
    if maps_shape is not None:
        pix = 1
        for d in maps_shape[2:]:
            pix *= d
        if len(maps_shape) < 3 or (maps_shape[0], maps_shape[1], pix) != (slots.shape[0], c, p):
            raise ValueError("maps must be [%d, %d, ...] with %d pixels, got %s" % (slots.shape[0], c, p, tuple(maps_shape)))


def _check_linear(x, w_q, w_scale, bias, x_scale, slots, channels_first, out_dtype):
    _tensor("x", x, _FLOATS + (torch.int8,))
    _tensor("w_q", w_q, (torch.int8,), (2,))
    _tensor("w_scale", w_scale, (torch.float32,), (1,))
    o, k = w_q.shape
    if o < 1 or k < 1:
        raise ValueError("w_q is empty: %s" % (tuple(w_q.shape),))
    if o > 1 << 27:
        raise ValueError("w_q has %d outputs, at most 2^27 fit one launch" % o)
    if k > _lib.INT8_MAX_K:
        raise ValueError("w_q has %d channels, at most %d are summed exactly in 32 bits" % (k, _lib.INT8_MAX_K))
    if w_scale.shape[0] != o:
        raise ValueError("w_scale must have shape (%d,), got %s" % (o, tuple(w_scale.shape)))
    if bias is not None:
        _tensor("bias", bias, (torch.float32,), (1,))
        if bias.shape[0] != o:
            raise ValueError("bias must have shape (%d,), got %s" % (o, tuple(bias.shape)))
    if out_dtype not in _FLOATS:
        raise TypeError("out_dtype must be float32, bfloat16 or float16, got %s" % (out_dtype,))
    if x.dtype != torch.int8:
        if x_scale is not None or slots is not None:
            raise ValueError("x_scale and slots go with 8-bit x; floating x is quantised by the call")
        if x.dim() < (3 if channels_first else 1):
            raise ValueError("x must be %s, got %s" % ("[B, K, ...]" if channels_first else "[..., K]", tuple(x.shape)))
        kx = x.shape[1 if channels_first else -1]
    else:
        if x_scale is None:
            raise ValueError("8-bit x needs its x_scale")
        _tensor("x_scale", x_scale, (torch.float32,))
        if x.dim() < 1 or tuple(x_scale.shape) != tuple(x.shape[:-1]):
            raise ValueError("x_scale must have the shape of x without its channels, got %s for x %s" % (tuple(x_scale.shape), tuple(x.shape)))
        if (slots is not None or channels_first) and x.dim() != 3:
            raise ValueError("with slots or channels_first, 8-bit x must be [n, P, K], got %s" % (tuple(x.shape),))
        if slots is not None:
            _tensor("slots", slots, (torch.int64,), (1,))
            if x.shape[0] < 1:
                raise ValueError("slots are given but x is empty: %s" % (tuple(x.shape),))
        kx = x.shape[-1]
    if kx != k:
        raise ValueError("x has %d channels, w_q has %d" % (kx, k))


# ---- layout --------------------------------------------------------------------------------------------------------------------
def _maps3(t):
    """[B, C, ...] -> [B, C, P] with contiguous pixels (a copy only where the strides need it)."""
    t = t.reshape(t.shape[0], t.shape[1], -1) if t.numel() else t.reshape(t.shape[0], t.shape[1], _count(t.shape[2:]))
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _count(dims):
    n = 1
    for d in dims:
        n *= d
    return n


def _rows3(t):
    """[..., K] -> [b, n, K] with contiguous channels."""
    k = t.shape[-1]
    if t.dim() == 3:
        pass
    elif t.dim() == 2:
        t = t.unsqueeze(0)
    else:
        t = t.reshape(1, _count(t.shape[:-1]), k)
    return t if t.stride(2) == 1 or k == 1 else t.contiguous()


def _one_entry(t):
    """Rows [b, n, K] as [1, b n, K] where the entries stand one behind the other: which kernel takes them goes by their number, not by how
    they are counted."""
    b, n, k = t.shape
    if b <= 1 or n < 1 or not (n == 1 or t.stride(0) == n * t.stride(1)):
        return t
    return t.as_strided((1, b * n, k), (0, t.stride(0) if n == 1 else t.stride(1), t.stride(2)))


def _pitched(q):
    """8-bit rows [b, n, K] as a product reads them: on 16-byte boundaries, readable to the next multiple of 16."""
    b, n, k = q.shape
    k16 = row_pitch(k, ROW_ALIGN)
    st = q.stride()
    ok = (st[2] == 1 or k == 1) and (n == 1 or (st[1] % ROW_ALIGN == 0 and st[1] >= k16)) and (b == 1 or st[0] % ROW_ALIGN == 0) and \
        q.data_ptr() % ROW_ALIGN == 0
    if ok:
        last = q.storage_offset() + (b - 1) * st[0] + (n - 1) * st[1] + k16
        ok = last <= q.untyped_storage().nbytes()
    if ok:
        return q
    out = empty_rows(b, n, k, device=q.device)
    out.copy_(q)
    return out


def _stride(t, d, other):
    return int(t.stride(d)) if t.shape[d] > 1 else int(other)


def _rows_problem(x3, channels_first, q, scale, slots=None):
    p = _lib.GnrRowsProblem()
    p.dtype, p.channels_first = _DTYPE[x3.dtype], int(channels_first)
    p.batch, p.channels, p.n_pix = x3.shape[0], x3.shape[1 if channels_first else 2], x3.shape[2 if channels_first else 1]
    p.x, p.x_batch, p.x_stride = x3.data_ptr(), int(x3.stride(0)), int(x3.stride(1))
    p.q, p.q_batch, p.q_pitch = q.data_ptr(), int(q.stride(0)), _stride(q, 1, row_pitch(q.shape[2]))
    p.scale, p.scale_batch = scale.data_ptr(), int(scale.stride(0))
    if slots is not None:
        p.slots, p.n_slots = slots.data_ptr(), q.shape[0]
    return p


def _call(fn, p, dev, *more):
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(getattr(lib, fn)(C.byref(p), *more, _stream_ptr(dev)), lib)


# ---- the operators -------------------------------------------------------------------------------------------------------------
def quantize_rows(x, channels_first: bool = False) -> QuantizedRows:
    """x [..., K] -> q [..., K], scale [...]; ``channels_first``: maps [B, K, ...] -> q [B, P, K], scale [B, P]."""
    _no_grad("quantize_rows", x)
    ext = _torch_ext.active()
    if ext is not None:
        try:
            return QuantizedRows(*ext.quantize_rows(x, bool(channels_first)))
        except (RuntimeError, TypeError) as e:
            _check_quantize(x, channels_first)
            raise _as_gnr(e) from e
    _check_quantize(x, channels_first)
    x3 = _maps3(x) if channels_first else _rows3(x)
    b, n, k = (x3.shape[0], x3.shape[2], x3.shape[1]) if channels_first else x3.shape
    q = empty_rows(b, n, k, device=x.device)
    scale = torch.empty(b, n, dtype=torch.float32, device=x.device)
    if x3.numel():
        _call("gnr_quantize_rows", _rows_problem(x3, channels_first, q, scale), x.device)
    if channels_first:
        return QuantizedRows(q, scale)
    return QuantizedRows(_unflatten(q, x.shape[:-1], k), scale.reshape(x.shape[:-1]))


def quantize_rows_into(x, q, scale) -> None:
    """``quantize_rows`` of x [N, K] into q int8 [N, K] and scale float32 [N] that the caller owns."""
    _no_grad("quantize_rows_into", x, scale)
    _check_quantize(x, False)
    _check_cache(q.unsqueeze(0), scale.unsqueeze(0), torch.empty(0, dtype=torch.int64), None)
    _one_device(x=x, q=q, scale=scale)
    if x.dim() != 2 or x.shape != q.shape:
        raise ValueError("x and q must be [N, K], got %s and %s" % (tuple(x.shape), tuple(q.shape)))
    x3 = _rows3(x)
    _call("gnr_quantize_rows", _rows_problem(x3, False, q.unsqueeze(0), scale.unsqueeze(0)), x.device)


def _unflatten(q, lead, k):
    pitch = row_pitch(k)
    strides, s = [], pitch
    for d in reversed(lead):
        strides.append(s)
        s *= d
    return q.as_strided(tuple(lead) + (k,), tuple(reversed(strides)) + (1,))


def _as_gnr(e):
    if isinstance(e, torch.cuda.OutOfMemoryError) or isinstance(e, TypeError):
        return e
    return _lib.GnrError(str(e).split("\n")[0])


def _check_quantize(x, channels_first):
    _tensor("x", x, _FLOATS)
    if x.dim() < (3 if channels_first else 1):
        raise ValueError("x must be %s, got %s" % ("[B, K, ...]" if channels_first else "[..., K]", tuple(x.shape)))
    if x.shape[1 if channels_first else -1] < 1:
        raise ValueError("x has no channels: %s" % (tuple(x.shape),))
    _one_device(x=x)


def write_featmaps(q, scale, slots, maps) -> None:
    """maps [B, C, P] (or [B, C, H, W]) go as 8-bit rows into slots[b] of the cache q int8 [n, P, C], scale float32 [n, P].

    ``slots``: int64 [B] on the device, not read by the host.  A negative slot is padding and a slot >= n a mistake: neither is
    written.  Of several maps with the same slot the last one stays.  Every other byte of the cache is left as it was."""
    _no_grad("write_featmaps", maps, scale)
    ext = _torch_ext.active()
    if ext is not None:
        try:
            ext.write_featmaps(q, scale, slots, maps)
            return
        except (RuntimeError, TypeError) as e:
            _check_write(q, scale, slots, maps)
            raise _as_gnr(e) from e
    _check_write(q, scale, slots, maps)
    m = _maps3(maps)
    if m.numel():
        slots = slots.contiguous()
        _call("gnr_quantize_rows", _rows_problem(m, True, q, scale, slots), q.device)


def _check_write(q, scale, slots, maps):
    _tensor("maps", maps, _FLOATS)
    _check_cache(q, scale, slots, maps.shape)
    _one_device(q=q, scale=scale, slots=slots, maps=maps)


def read_featmaps(q, scale, slots, out_dtype=torch.float32):
    """slots int64 [B] of the cache -> maps [B, C, P].  A negative slot reads as zeros, a slot >= n as NaN."""
    _no_grad("read_featmaps", scale)
    ext = _torch_ext.active()
    if ext is not None and out_dtype in _FLOATS:
        try:
            return ext.read_featmaps(q, scale, slots, _DTYPE[out_dtype])
        except (RuntimeError, TypeError) as e:
            _check_read(q, scale, slots, out_dtype)
            raise _as_gnr(e) from e
    _check_read(q, scale, slots, out_dtype)
    out = torch.empty(slots.shape[0], q.shape[2], q.shape[1], dtype=out_dtype, device=q.device)
    if out.numel():
        slots = slots.contiguous()
        _call("gnr_read_rows", _rows_problem(out, True, q, scale, slots), q.device)
    return out


def _check_read(q, scale, slots, out_dtype):
    if out_dtype not in _FLOATS:
        raise TypeError("out_dtype must be float32, bfloat16 or float16, got %s" % (out_dtype,))
    _check_cache(q, scale, slots, None)
    _one_device(q=q, scale=scale, slots=slots)


def int8_linear(x, w_q, w_scale, bias=None, *, x_scale=None, slots=None, leaky: bool = False, channels_first: bool = False,
                out_dtype=torch.float32):
    """act(x w^T + bias) with 8-bit operands: y(n, o) = act((sum_k xq(n,k) wq(o,k)) * x_scale(n) * w_scale(o) + bias(o)).

    x        float rows [..., K] -> y [..., O];  with ``channels_first`` float maps [B, K, ...] -> y [B, O, ...] (a 1x1 convolution).
             Each row is quantised by the call (``quantize_rows``).
             int8 rows [..., K] with ``x_scale`` [...] -> y [..., O];  with ``channels_first`` rows [B, P, K] -> y [B, O, P].
             With ``slots`` (int64 [B], on the device) x is a cache [n, P, K]: entry b is slot slots[b]; a negative slot counts as
             zero rows, a slot >= n gives NaN.
    w_q      int8 [O, K], w_scale float32 [O]: ``quantize_rows(weight)``.   bias: float32 [O] or None.
    leaky    LeakyReLU(0.2) behind the bias.
    The sum is exact (K <= 131071), the epilogue fp32, y is rounded once to ``out_dtype``."""
    _no_grad("int8_linear", x, w_scale, bias, x_scale)
    ext = _torch_ext.active()
    if ext is not None and out_dtype in _FLOATS:
        try:
            return ext.int8_linear(x, w_q, w_scale, bias, x_scale, slots, bool(leaky), bool(channels_first), _DTYPE[out_dtype])
        except (RuntimeError, TypeError) as e:
            _check_linear(x, w_q, w_scale, bias, x_scale, slots, channels_first, out_dtype)
            _one_device(x=x, w_q=w_q, w_scale=w_scale, bias=bias, x_scale=x_scale, slots=slots)
            raise _as_gnr(e) from e
    _check_linear(x, w_q, w_scale, bias, x_scale, slots, channels_first, out_dtype)
    _one_device(x=x, w_q=w_q, w_scale=w_scale, bias=bias, x_scale=x_scale, slots=slots)
    o, k = w_q.shape
    dev = x.device
    w = _pitched(w_q.unsqueeze(0))
    ws_c, b_c = w_scale.contiguous(), None if bias is None else bias.contiguous()
    p = _lib.GnrInt8Problem()
    p.x_type, p.y_type, p.leaky, p.k, p.o = _DTYPE[x.dtype], _DTYPE[out_dtype], int(bool(leaky)), k, o
    p.y_channels_first = int(bool(channels_first))
    keep = [w, ws_c, b_c]
    if x.dtype == torch.int8:
        xr = _pitched(_rows3(x))
        xs = x_scale.reshape(xr.shape[:2]) if x.dim() != 3 else x_scale
        xs = xs if xs.stride(1) == 1 or xs.shape[1] == 1 else xs.contiguous()
        b, n = xr.shape[:2]
        p.x_scale, p.x_scale_batch = xs.data_ptr(), int(xs.stride(0))
        p.x_batch, p.x_stride = _stride(xr, 0, 0), _stride(xr, 1, row_pitch(k))
        if slots is not None:
            sl = slots.contiguous()
            p.slots, p.n_slots = sl.data_ptr(), b
            b = sl.shape[0]
            keep.append(sl)
        keep += [xr, xs]
        lead = (b, n) if slots is not None else tuple(x.shape[:-1])
        shape = (b, o, n) if channels_first else lead + (o,)
    elif channels_first:
        xr = _maps3(x)
        b, n = xr.shape[0], xr.shape[2]
        p.x_channels_first, p.x_batch, p.x_stride = 1, int(xr.stride(0)), int(xr.stride(1))
        shape = (b, o) + tuple(x.shape[2:])
        keep.append(xr)
    else:
        xr = _one_entry(_rows3(x))
        b, n = xr.shape[:2]
        p.x_batch, p.x_stride = int(xr.stride(0)), int(xr.stride(1))
        shape = tuple(x.shape[:-1]) + (o,)
        keep.append(xr)
    y = torch.empty(shape, dtype=out_dtype, device=dev)
    if not y.numel():
        return y
    p.batch, p.n_pix, p.x, p.w, p.w_pitch = b, n, xr.data_ptr(), w.data_ptr(), _stride(w, 1, row_pitch(k))
    p.w_scale, p.bias, p.y = ws_c.data_ptr(), None if b_c is None else b_c.data_ptr(), y.data_ptr()
    lib = _lib.load()
    need = lib.gnr_int8_linear_workspace_bytes(C.byref(p))
    if need == 0:
        _lib.check(1, lib)
    ws = torch.empty(int(need), dtype=torch.uint8, device=dev)
    _call("gnr_int8_linear", p, dev, C.c_void_p(ws.data_ptr()), ws.numel())
    return y


class FeatureMapCache:
    """``n_slots`` feature maps of ``channels`` x ``n_pix`` kept as 8-bit rows on ``device`` (275 bytes a pixel at 258 channels).

    Slots are the caller's to hand out.  A slot that was never written reads as NaN.  Slots are given as an int, a sequence (checked on
    the host) or an int64 tensor on the device (not read by the host: see ``write_featmaps`` for slots outside the cache)."""

    def __init__(self, n_slots: int, channels: int = 258, n_pix: int = 4096, device="cuda"):
        if n_slots < 1 or channels < 1 or n_pix < 1:
            raise ValueError("FeatureMapCache(%r slots, %r channels, %r pixels): all must be >= 1" % (n_slots, channels, n_pix))
        self.q = torch.zeros(n_slots, n_pix, row_pitch(channels, ROW_ALIGN), dtype=torch.int8, device=device)[..., :channels]
        self.scale = torch.full((n_slots, n_pix), float("nan"), dtype=torch.float32, device=device)

    @property
    def n_slots(self):
        return self.q.shape[0]

    def slots(self, slots) -> torch.Tensor:
        if torch.is_tensor(slots):
            return slots
        slots = [operator.index(s) for s in ([slots] if hasattr(slots, "__index__") else slots)]
        for s in slots:
            if s >= self.n_slots:
                raise IndexError("slot %d of a cache of %d" % (s, self.n_slots))
        return torch.tensor(slots, dtype=torch.int64, device=self.q.device)

    def write(self, slots, maps) -> None:
        write_featmaps(self.q, self.scale, self.slots(slots), maps)

    def read(self, slots, out_dtype=torch.float32):
        return read_featmaps(self.q, self.scale, self.slots(slots), out_dtype)

    def linear(self, slots, w_q, w_scale, bias=None, **kw):
        """``int8_linear`` on the cached rows, without reading them back."""
        return int8_linear(self.q, w_q, w_scale, bias, x_scale=self.scale, slots=self.slots(slots), **kw)
