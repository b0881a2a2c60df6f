"""Microscaled 4-bit and 8-bit tensors: quantisation, the product of two of them, and the RMS norm that writes them.

A :class:`MicroscaledTensor` keeps its last dimension in blocks of 32 elements that share one power of two.  Format
``"mxfp4"`` has e2m1 elements (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), ``"mxfp8"`` e4m3 elements (up to 448);
a block's scale is ``2^(c - 127)`` with ``c - 127 = floor(log2 max|x|) - 2`` (4 bits) or ``- 8`` (8 bits), at least
-127.  Elements are rounded to nearest even and saturated.  A zero block has ``c = 0``; a block that holds a NaN or an
infinity has ``c = 255`` and reads as NaN throughout.

Like the other ops of this package the functions take CUDA tensors, launch on the stream that is current at call time
on the tensors' device, and record no autograd graph; there is no CPU path.
"""
import math

import torch
from torch import nn

from . import _cabi as C

BLOCK = 32
FORMATS = {"mxfp4": 4, "mxfp8": 8}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _format(name, what="format"):
    if name not in FORMATS:
        raise NotImplementedError('%s must be "mxfp4" or "mxfp8", got %r' % (what, name))
    return FORMATS[name]


def _dtype(dtype, what):
    if dtype not in _DTYPES:
        raise NotImplementedError("nesgpu_b200: %s must have dtype float32, bfloat16 or float16, got %s" % (what, dtype))
    return _DTYPES[dtype]


def _pitches(cols, format):
    """Bytes of codes and of scales per row: rows are padded to whole groups of 128 elements."""
    groups = -(-cols // 128)
    return groups * (64 if format == "mxfp4" else 128), groups * 4


_current_device, _raw_stream = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream


def _launch(name, device, *args):
    """Calls an entry point on ``device`` and the stream that is current there."""
    index = device.index
    if index == _current_device():
        return C.call(name, *args, _raw_stream(index))
    with torch.cuda.device(device):
        return C.call(name, *args, _raw_stream(index))


def _same_device(device, name, t):
    if t is not None and t.device != device:
        raise RuntimeError("nesgpu_b200: %s is on %s, expected %s" % (name, t.device, device))


class MicroscaledTensor:
    """Codes and scales of a ``(..., cols)`` tensor.

    ``codes`` is ``(rows, 64 * G)`` uint8 for ``"mxfp4"`` (two elements to a byte, the even column in the low half)
    or ``(rows, 128 * G)`` for ``"mxfp8"``, ``scales`` ``(rows, 4 * G)`` uint8, with ``G = ceil(cols / 128)``; both
    contiguous CUDA tensors whose padding is zero.  ``shape`` gives the leading dimensions if there are several (their
    product is ``rows``).  The object refers to the tensors it is given."""

    __slots__ = ("codes", "scales", "rows", "cols", "format", "_lead")

    def __init__(self, codes, scales, cols, format="mxfp4", shape=None):
        _format(format)
        cols = int(cols)
        if cols < 1:
            raise RuntimeError("a microscaled tensor needs at least one column")
        codes = C.require_cuda(codes, "codes", torch.uint8)
        scales = C.require_cuda(scales, "scales", torch.uint8)
        _same_device(codes.device, "scales", scales)
        pitch, spitch = _pitches(cols, format)
        rows = codes.shape[0] if codes.dim() else 0
        if codes.shape != (rows, pitch) or scales.shape != (rows, spitch):
            raise RuntimeError("codes and scales of %d columns in %s must be (rows, %d) and (rows, %d), got %s and %s"
                               % (cols, format, pitch, spitch, tuple(codes.shape), tuple(scales.shape)))
        if codes.data_ptr() % 32:                # the kernels read codes in aligned 16- and 32-byte pieces
            codes = codes.clone()
        if scales.data_ptr() % 4:
            scales = scales.clone()
        lead = (rows,) if shape is None else tuple(int(s) for s in shape)
        if math.prod(lead) != rows:
            raise RuntimeError("leading dimensions %s do not match %d rows" % (lead, rows))
        self.codes, self.scales, self.rows, self.cols, self.format, self._lead = codes, scales, rows, cols, format, lead

    @property
    def shape(self):
        return torch.Size((*self._lead, self.cols))

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return "MicroscaledTensor(shape=%s, format=%s, device=%s)" % (tuple(self.shape), self.format, self.device)

    def _view(self, t, width):
        """The first ``width`` columns of a row-major byte matrix, with this tensor's leading dimensions."""
        if t.shape[1] != width:
            t = t.narrow(1, 0, width)
        return t if len(self._lead) == 1 else t.unflatten(0, self._lead)

    def block_scales(self):
        """``(..., ceil(cols / 32))`` scales as ``torch.float8_e8m0fnu`` (a view)."""
        return self._view(self.scales, -(-self.cols // BLOCK)).view(torch.float8_e8m0fnu)

    def elements(self):
        """``(..., cols)`` element values before the scale, as ``torch.float8_e4m3fn``: a view for ``"mxfp8"``,
        unpacked for ``"mxfp4"`` (every e2m1 value is an e4m3 value)."""
        if self.format == "mxfp8":
            return self._view(self.codes, self.cols).view(torch.float8_e4m3fn)
        codes = self.codes
        out = codes.new_empty((*self._lead, self.cols), dtype=torch.float8_e4m3fn)
        _launch("nes_mx_elements", codes.device, codes.data_ptr(), out.data_ptr(), self.rows, self.cols)
        return out

    def dequantize(self, dtype=torch.float32):
        """The values ``element * scale`` (exact in fp32; rounded to nearest even in bfloat16 and float16)."""
        kind = _dtype(dtype, "the result")
        out = self.codes.new_empty(self.shape, dtype=dtype)
        _launch("nes_mx_dequantize", self.codes.device, self.codes.data_ptr(), self.scales.data_ptr(), out.data_ptr(), kind,
                self.rows, self.cols, FORMATS[self.format])
        return out


def _empty(x, rows, cols, format):
    """Uninitialised blocks for ``rows`` rows, with the leading dimensions and on the device of ``x``."""
    pitch, spitch = _pitches(cols, format)
    q = MicroscaledTensor.__new__(MicroscaledTensor)
    q.codes = x.new_empty((rows, pitch), dtype=torch.uint8)
    q.scales = x.new_empty((rows, spitch), dtype=torch.uint8)
    q.rows, q.cols, q.format, q._lead = rows, cols, format, x.shape[:-1]
    return q


def _aligned(t):
    """``t`` at an address that is a multiple of 16 bytes (a copy if it starts inside an allocation)."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _rows(t, name):
    """A contiguous CUDA tensor of a supported type with at least one column, and its number of rows."""
    t = C.require_cuda(t, name)
    _dtype(t.dtype, name)
    if t.dim() == 0 or t.shape[-1] == 0:
        raise RuntimeError("%s needs at least one column, got shape %s" % (name, tuple(t.shape)))
    return t, t.numel() // t.shape[-1]


def quantize(input, format="mxfp4"):
    """``(..., cols)`` float32 / bfloat16 / float16 -> :class:`MicroscaledTensor`."""
    kind = _format(format)
    x, rows = _rows(input, "input")
    cols = x.shape[-1]
    q = _empty(x, rows, cols, format)
    _launch("nes_mx_quantize", x.device, x.data_ptr(), _DTYPES[x.dtype], q.codes.data_ptr(), q.scales.data_ptr(), rows,
            cols, kind)
    return q


def linear(input, weight, bias=None, activations="mxfp8", dtype=None, out=None):
    """``y = x W^T + b`` with both operands microscaled: ``weight`` a :class:`MicroscaledTensor` of ``(out, in)``,
    ``input`` either one of ``(..., in)`` or a plain tensor, which is quantised to ``activations`` on the way.

    Products are accumulated in fp32 and rounded once to ``dtype`` (default: the type of a plain input, float32 for a
    microscaled one).  8-bit activations take weights of either format, 4-bit activations 4-bit weights.  ``out``
    receives the result if given (contiguous, of the result's type and number of elements)."""
    if not isinstance(weight, MicroscaledTensor) or len(weight._lead) != 1:
        raise RuntimeError("weight must be a MicroscaledTensor of (out_features, in_features)")
    out_features, in_features = weight.rows, weight.cols
    x_scales, x_kind = None, 0
    if isinstance(input, MicroscaledTensor):
        x, rows, activations, default = input.codes, input.rows, input.format, torch.float32
        x_scales, lead, cols = input.scales.data_ptr(), input._lead, input.cols
    else:
        x, rows = _rows(input, "input")
        x_kind, default, lead, cols = _DTYPES[x.dtype], x.dtype, x.shape[:-1], x.shape[-1]
    if dtype is None:
        dtype = default if out is None else out.dtype
    x_format, y_kind = _format(activations, "activations"), _dtype(dtype, "the result")
    device = x.device
    if cols != in_features:
        raise RuntimeError("expected last dimension %d, got %d" % (in_features, cols))
    _same_device(device, "weight", weight.codes)
    if bias is not None:
        bias = C.require_cuda(bias, "bias", torch.float32)
        if bias.shape != (out_features,):
            raise RuntimeError("bias must have shape (%d,), got %s" % (out_features, tuple(bias.shape)))
        _same_device(device, "bias", bias)
    y = out
    if out is None:
        y = x.new_empty((*lead, out_features), dtype=dtype)
    elif out.device != device or out.dtype != dtype or not out.is_contiguous() or out.numel() != rows * out_features:
        raise RuntimeError("out must be a contiguous %s tensor of %d elements on %s" % (dtype, rows * out_features, device))
    buf, nbytes = None, 0
    if x_scales is None:
        nbytes = C.call("nes_mx_linear_fwd_scratch_bytes", rows, out_features, in_features, x_format)
        if nbytes:      # a buffer of this call's own: calls captured into different graphs share nothing
            buf = x.new_empty(nbytes, dtype=torch.uint8)
    _launch("nes_mx_linear_fwd", device, x.data_ptr(), x_scales, x_kind, x_format, weight.codes.data_ptr(),
            weight.scales.data_ptr(), FORMATS[weight.format], C.ptr(bias), y.data_ptr(), y_kind, rows, out_features,
            in_features, C.ptr(buf), nbytes)
    return y


def rms_norm(input, weight=None, eps=1e-6, residual=None, noise=None, antithetic=False, output=None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, with ``h = input + residual``.

    ``weight`` is a float32 gain per column (ones if None).  ``residual`` has the input's shape and type; with it the
    call returns ``(y, h)``, ``h`` rounded to that type (``y`` is computed from the unrounded sum).  ``noise``
    ``(members, cols)`` float32 adds ``noise[d]`` to the gain of the rows ``r * members + d`` (its negative for the
    second half of the repeats with ``antithetic``).  ``output`` is None for a ``y`` of the input's type, or
    ``"mxfp8"`` / ``"mxfp4"`` for a :class:`MicroscaledTensor`."""
    x, rows = _rows(input, "input")
    cols, device = x.shape[-1], x.device
    kind = 0 if output is None or output == x.dtype else _format(output, "output")
    if not eps >= 0:
        raise RuntimeError("eps must not be negative, got %r" % (eps,))
    h, members = None, 0
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != x.shape:
            raise RuntimeError("residual must have the input's shape %s" % (tuple(x.shape),))
        residual = C.require_cuda(residual, "residual", x.dtype)
        _same_device(device, "residual", residual)
        h = torch.empty_like(x)
    if weight is not None:
        weight = C.require_cuda(weight, "weight", torch.float32)
        if weight.shape != (cols,):
            raise RuntimeError("weight must have shape (%d,), got %s" % (cols, tuple(weight.shape)))
        _same_device(device, "weight", weight)
    if noise is not None:
        noise = C.require_cuda(noise, "noise", torch.float32)
        members = noise.shape[0] if noise.dim() else 0
        if not members or noise.shape != (members, cols):
            raise RuntimeError("noise must have shape (members, %d), got %s" % (cols, tuple(noise.shape)))
        if rows % members:
            raise RuntimeError("batch size %d is not a multiple of directions %d" % (rows, members))
        _same_device(device, "noise", noise)
    if kind:
        y = _empty(x, rows, cols, output)
        data, scales = y.codes.data_ptr(), y.scales.data_ptr()
    else:
        y = torch.empty_like(x)
        data, scales = y.data_ptr(), None
    x, residual, weight, noise = _aligned(x), _aligned(residual), _aligned(weight), _aligned(noise)
    _launch("nes_rms_norm_fwd", device, x.data_ptr(), C.ptr(residual), C.ptr(h), C.ptr(weight), C.ptr(noise), data,
            scales, rows, cols, members, 1 if antithetic else 0, _DTYPES[x.dtype], kind, eps)
    return y if residual is None else (y, h)


class MicroscaledLinear(nn.Module):
    """A linear layer whose weight is kept microscaled, for evaluating or serving a trained model: the buffers
    ``weight_codes`` / ``weight_scales`` replace the fp32 parameter.  Build it with :meth:`from_linear`."""

    def __init__(self, in_features, out_features, bias=True, format="mxfp4", activations="mxfp8", device=None):
        super().__init__()
        _format(format)
        if FORMATS[format] > _format(activations, "activations"):
            raise NotImplementedError("4-bit activations need 4-bit weights")
        self.in_features, self.out_features = in_features, out_features
        self.format, self.activations = format, activations
        pitch, spitch = _pitches(in_features, format)
        self.register_buffer("weight_codes", torch.zeros((out_features, pitch), dtype=torch.uint8, device=device))
        self.register_buffer("weight_scales", torch.zeros((out_features, spitch), dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear, format="mxfp4", activations="mxfp8"):
        """Quantises the weight of any ``nn.Linear`` (the perturbed layers among them) as it is now."""
        q = quantize(linear.weight.detach(), format)
        layer = cls(linear.in_features, linear.out_features, linear.bias is not None, format, activations, q.device)
        layer.weight_codes.copy_(q.codes)
        layer.weight_scales.copy_(q.scales)
        if linear.bias is not None:
            layer.bias.copy_(linear.bias.detach())
        return layer

    @property
    def weight(self):
        return MicroscaledTensor(self.weight_codes, self.weight_scales, self.in_features, self.format)

    def forward(self, input, dtype=None):
        return linear(input, self.weight, self.bias, self.activations, dtype)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s, format=%s, activations=%s" % (
            self.in_features, self.out_features, self.bias is not None, self.format, self.activations)
