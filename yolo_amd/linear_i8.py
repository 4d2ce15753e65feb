"""Linear layers and 1x1 convolutions in 8-bit integers, with one scale per row of the input (pixel, token) and one per
output channel (y3_linear_i8, include/yolo3hip.h):

    layer = Int8Linear(weight, bias, leaky=True)      weight [n, k] float, or int8 with scale=[n]
    y = layer(x)                                      x [..., k] float32 / bfloat16: rows are quantised on the way
    rows = quantize_rows(x)                           once, for several layers:
    y1, y2 = layer1(rows.values, scale=rows.scale), layer2(rows.values, scale=rows.scale)

    y[m, n] = act(s[m] t[n] sum_k q[m, k] w[n, k] + bias[n]),
    q = round_half_even(x * (127 * (1 / a))),  s = a / 127,  a = max(max_k |x_k|, 127 * 2^-126)   (in fp32)

The sum is exact, so a row's result does not depend on the rows beside it.  A row with a NaN or an infinity gives NaN.
`Network(..., int8=True)` runs its 1x1 convolutions this way.  Calls are asynchronous on the current stream of the
layer's device; nothing is kept from one call for the next, so calls on several streams and in HIP graphs are independent.
A layer waits for its weights to be laid out before it is returned, so any stream may call it; one that is made inside a
capture holds them after the first replay.
There is no gradient (the package is inference only): tensors that require one, or carry a tangent, are refused.
"""
import collections
import ctypes
import operator

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib

_CODES = {torch.float32: _lib.Y3_F32, torch.bfloat16: _lib.Y3_BF16, torch.int8: _lib.Y3_I8}
Int8Rows = collections.namedtuple("Int8Rows", "values scale")
MAX_K, MAX_N = 131071, 1 << 24          # what the library takes; its own check sees 32 bits of a size only

# the current stream's handle, without making a Stream object (1.7 us of a call that takes 6)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _rows_of(x, k, name):
    """x [..., k] as a matrix whose rows lie at one stride and whose elements are adjacent (copied only if they are not)."""
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError("%s: last dimension must be %d, got shape %r" % (name, k, tuple(x.shape)))
    if x.dim() != 2:
        x = x.reshape(-1, k)
    if (k > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < k):
        x = x.contiguous()
    return x


def _refuse_gradient(t, name, what):
    """Neither direction of differentiation goes through the kernels: nothing is dropped without a word.  (Where every call
    passes, its callers look at requires_grad and the level themselves first: 0.1 us each.)"""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient: %s has none (use torch.no_grad())" % (name, what))
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError("%s carries a tangent: %s has no forward derivative" % (name, what))


def _check_input(x, name):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("%s must be a tensor on the GPU" % name)
    if x.requires_grad or _forward_ad._current_level >= 0:
        _refuse_gradient(x, name, "the 8-bit product")


def _eight_bit_rows(x, n):
    """8-bit rows and their pitch as y3_linear_i8 takes them.  Rows on 16 bytes are read up to a multiple of 16, which has to
    be there; others are read as they are, or copied where the product takes far longer than a copy (the kernel for many
    rows and channels needs them on 16 bytes: 8192 x 8192 -> 8192 in half the time)."""
    rows, k = x.shape
    pitch = (k + 15) // 16 * 16
    ld = x.stride(0) if rows > 1 else pitch
    aligned = x.data_ptr() % 16 == 0 and ld % 16 == 0 and ld >= pitch
    if aligned and (k == pitch or x.storage_offset() + (rows - 1) * ld + pitch <= x.untyped_storage().nbytes()):
        return x, ld
    ld = x.stride(0) if rows > 1 else k
    if not (rows > 1 and aligned) and (k < 512 or rows * n < 1 << 23):
        return x, ld
    q = torch.empty((rows, pitch), dtype=torch.int8, device=x.device)
    _lib.check(_lib.load().y3_quantize_rows_i8(_lib.Y3_I8, x.data_ptr(), rows, k, ld, q.data_ptr(), pitch, None,
                                               _stream_of(x.device.index)))
    return q, pitch


def quantize_rows(x):
    """x [..., k] float32 / bfloat16 -> Int8Rows(values int8 [..., k], scale float32 [...]): values * scale stands for x.
    The values are a view of rows padded to 16 bytes, which is how Int8Linear reads them without a copy."""
    _check_input(x, "x")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("quantize_rows: float32 or bfloat16, got %s" % x.dtype)
    lead, k = x.shape[:-1], x.shape[-1] if x.dim() else 0
    if k > MAX_K:
        raise ValueError("quantize_rows: rows of %d, at most %d" % (k, MAX_K))
    m = _rows_of(x, k, "x")
    rows, pitch = m.shape[0], (k + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=torch.int8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().y3_quantize_rows_i8(_CODES[x.dtype], m.data_ptr(), rows, k, m.stride(0) if rows > 1 else k,
                                                   q.data_ptr(), pitch, s.data_ptr(), _stream_of(x.device.index)))
    return Int8Rows(q[:, :k].view(lead + (k,)) if len(lead) == 1 else q.view(lead + (pitch,))[..., :k], s.view(lead))


class Int8Linear(object):
    """weight [n, k]: float32 / bfloat16 (each row quantised here), or int8 with its scale float32 [n].  bias [n] or None.
    out_dtype torch.bfloat16 (default) or torch.float32; leaky: leaky-ReLU (alpha 0.1) behind the bias.
    The attributes are read-only: descriptors and pointers that calls use are kept from the first one on."""

    n, k, device, leaky, out_dtype, bias, scale = (
        property(operator.attrgetter("_" + name)) for name in ("n", "k", "device", "leaky", "out_dtype", "bias", "scale"))

    def __init__(self, weight, bias=None, scale=None, leaky=False, out_dtype=torch.bfloat16, device=None):
        weight = torch.as_tensor(weight)
        if device is None:
            device = weight.device if weight.is_cuda else torch.device("cuda", torch.cuda.current_device())
        self._device = torch.device(device)
        if self._device.type != "cuda":
            raise ValueError("Int8Linear needs a GPU, got device %s" % self._device)
        if self._device.index is None:
            self._device = torch.device("cuda", torch.cuda.current_device())
        if weight.dim() != 2 or weight.dtype not in _CODES:
            raise ValueError("weight must be [n, k] float32, bfloat16 or int8, got %s %r" % (weight.dtype, tuple(weight.shape)))
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("out_dtype must be torch.bfloat16 or torch.float32, got %s" % out_dtype)
        if (weight.dtype == torch.int8) != (scale is not None):
            raise ValueError("scale goes with an int8 weight, and only with one")
        for t, name in ((weight, "weight"), (bias, "bias"), (scale, "scale")):
            if isinstance(t, torch.Tensor):
                _refuse_gradient(t, name, "the 8-bit product")
        self._n, self._k = int(weight.shape[0]), int(weight.shape[1])
        if self._n > MAX_N or self._k > MAX_K:
            raise ValueError("weight is %d x %d, at most %d x %d" % (self._n, self._k, MAX_N, MAX_K))
        self._leaky, self._out_dtype = bool(leaky), out_dtype
        lib = _lib.load()
        d = _lib.LinearI8Desc()
        d.k, d.n = self._k, self._n
        _lib.check(lib.y3_linear_i8_layout(ctypes.byref(d)))
        self._k_pad, self._n_pad = d.k_pad, d.n_pad
        weight = weight.detach().to(self._device).contiguous()

        def vector(v, what):
            v = torch.as_tensor(v).detach()
            if v.shape != (self._n,):
                raise ValueError("%s must have shape (%d,), got %r" % (what, self._n, tuple(v.shape)))
            # (a copy: the caller's tensor may change or be freed, like the weight it was given with)
            return torch.empty(self._n, dtype=torch.float32, device=self._device).copy_(v)

        self._bias = vector(bias, "bias") if bias is not None else None
        self._scale = vector(scale, "scale") if scale is not None else torch.empty(self._n, dtype=torch.float32, device=self._device)
        self._packed = torch.empty(self._k_pad * self._n_pad, dtype=torch.int8, device=self._device)
        with torch.cuda.device(self._device):
            _lib.check(lib.y3_linear_i8_pack(ctypes.byref(d), _CODES[weight.dtype], weight.data_ptr(), self._k,
                                             self._packed.data_ptr(), self._scale.data_ptr(), _stream_of(self._device.index)))
            # Later calls may be on any stream, and their callers may not know of this launch (a network packs while it
            # builds a plan): wait for it here, once.  In a capture the graph orders it before the calls that it holds.
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        self._bind()

    def _bind(self):
        """What calls keep: descriptors by shape, and this object's pointers."""
        self._descs = {}
        self._weights = (self._packed.data_ptr(), self._scale.data_ptr(), self._bias.data_ptr() if self._bias is not None else None)

    def __getstate__(self):                 # (copy, pickle: neither of them is the copy's)
        return {k: v for k, v in self.__dict__.items() if k not in ("_descs", "_weights")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    def _desc(self, key):
        """(descriptor, workspace bytes) of a call's shape."""
        code, rows, x_ld, out_ld = key
        d = _lib.LinearI8Desc()
        d.dtype, d.out_dtype, d.k, d.n, d.rows = code, _CODES[self._out_dtype], self._k, self._n, rows
        d.x_ld, d.out_ld, d.k_pad, d.n_pad = x_ld, out_ld, self._k_pad, self._n_pad
        d.flags = _lib.CONV_LEAKY if self._leaky else 0
        need = ctypes.c_int64(0)
        _lib.check(_lib.load().y3_linear_i8_workspace_bytes(ctypes.byref(d), ctypes.byref(need)))
        if len(self._descs) >= 256:         # shapes of a service come and go
            self._descs.clear()
        self._descs[key] = hit = (ctypes.byref(d), int(need.value))
        return hit

    def __call__(self, x, scale=None, out=None):
        """x [..., k] float32 / bfloat16, or int8 with scale float32 [...].  Returns [..., n] (in `out` if given)."""
        _check_input(x, "x")
        device = self._device
        if x.device != device:
            raise ValueError("x is on %s, the layer on %s" % (x.device, device))
        if device.index != torch.cuda.current_device():         # launches go to the current device
            with torch.cuda.device(device):
                return self(x, scale=scale, out=out)
        code = _CODES.get(x.dtype)
        if code is None:
            raise ValueError("x must be float32, bfloat16 or int8, got %s" % x.dtype)
        if (code == _lib.Y3_I8) != (scale is not None):
            raise ValueError("scale goes with int8 rows, and only with them")
        m = _rows_of(x, self._k, "x")
        rows = m.shape[0]
        shape = (rows, self._n) if m is x else x.shape[:-1] + (self._n,)
        if out is None:
            out = x.new_empty(shape, dtype=self._out_dtype)
            out_ld = self._n
        else:
            _refuse_gradient(out, "out", "the 8-bit product")
            if out.dtype != self._out_dtype or out.shape != shape or out.device != device:
                raise ValueError("out must be %s %r on %s" % (self._out_dtype, tuple(shape), device))
            flat = out.view(-1, self._n) if rows else out            # (a view: rows at one stride, or this raises)
            out_ld = flat.stride(0) if rows > 1 else self._n
            if (self._n > 1 and rows and flat.stride(1) != 1) or out_ld < self._n:
                raise ValueError("out must have adjacent elements in each row and rows that do not overlap")
        if rows == 0:
            return out
        scale_ptr = None
        if code == _lib.Y3_I8:
            if scale.dtype != torch.float32 or scale.device != device or scale.shape not in (x.shape[:-1], (rows,)):
                raise ValueError("scale must be float32 %r on %s" % (tuple(x.shape[:-1]), device))
            _refuse_gradient(scale, "scale", "the 8-bit product")
            scale = scale.contiguous()
            scale_ptr = scale.data_ptr()
            m, x_ld = _eight_bit_rows(m, self._n)
        else:
            x_ld = m.stride(0) if rows > 1 else self._k
        key = (code, rows, x_ld, out_ld)
        dref, need = self._descs.get(key) or self._desc(key)
        ws = x.new_empty(need, dtype=torch.uint8) if need else None
        w, ws_scale, b = self._weights
        rc = _lib.load().y3_linear_i8(dref, m.data_ptr(), scale_ptr, w, ws_scale, b, out.data_ptr(),
                                      ws.data_ptr() if need else None, need, _stream_of(device.index))
        if rc:
            _lib.check(rc)
        return out
