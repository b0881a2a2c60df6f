"""Microscaled 4-bit and 8-bit tensors: quantisation, the product of two of them, and the RMS norm that writes them.

A :class:`MicroscaledTensor` keeps its last dimension in blocks of 32 elements that share one power of two.  Format
``"mxfp4"`` has e2m1 elements (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), ``"mxfp8"`` e4m3 elements (up to 448);
a block's scale is ``2^(c - 127)`` with ``c - 127 = floor(log2 max|x|) - 2`` (4 bits) or ``- 8`` (8 bits), at least
-127.  Elements are rounded to nearest even and saturated.  A zero block has ``c = 0``; a block that holds a NaN or an
infinity has ``c = 255`` and reads as NaN throughout.

Like the other ops of this package the functions take CUDA tensors, launch on the stream that is current at call time
on the tensors' device, and record no autograd graph; there is no CPU path.
"""
import importlib
import math

import torch
from torch import nn

from . import _cabi  # noqa: F401  (loads the library that the extension module is linked with)


class _Unloaded:
    """Stands for the extension module until a call needs it: it is built for one PyTorch and one Python, on which the layers
    without microscaled calls do not depend."""

    def __getattr__(self, name):
        global _host
        try:
            module = importlib.import_module("._host", __package__)
        except ImportError as e:
            raise RuntimeError("nesgpu_b200: the extension module _host cannot be loaded (%s). Build it with `python -m "
                               "nesgpu_b200.build`; there is no fallback path." % e) from e
        _host = module
        return getattr(module, name)


_host = _Unloaded()

BLOCK = 32
FORMATS = {"mxfp4": 4, "mxfp8": 8}


def _format(name, what="format"):
    if name not in FORMATS:
        raise NotImplementedError('%s must be "mxfp4" or "mxfp8", got %r' % (what, name))
    return FORMATS[name]


def _pitches(cols, format):
    """Bytes of codes and of scales per row: rows are padded to whole groups of 128 elements."""
    groups = -(-cols // 128)
    return groups * (64 if format == "mxfp4" else 128), groups * 4


class MicroscaledTensor:
    """Codes and scales of a ``(..., cols)`` tensor.

    ``codes`` is ``(rows, 64 * G)`` uint8 for ``"mxfp4"`` (two elements to a byte, the even column in the low half)
    or ``(rows, 128 * G)`` for ``"mxfp8"``, ``scales`` ``(rows, 4 * G)`` uint8, with ``G = ceil(cols / 128)``; both
    contiguous CUDA tensors whose padding is zero.  ``shape`` gives the leading dimensions if there are several (their
    product is ``rows``).  The object refers to the tensors it is given."""

    __slots__ = ("codes", "scales", "rows", "cols", "format", "_lead")

    def __init__(self, codes, scales, cols, format="mxfp4", shape=None):
        self.codes, self.scales, rows = _host.blocks(codes, scales, cols, _format(format))
        lead = (rows,) if shape is None else tuple(int(s) for s in shape)
        if math.prod(lead) != rows:
            raise RuntimeError("leading dimensions %s do not match %d rows" % (lead, rows))
        self.rows, self.cols, self.format, self._lead = rows, cols, format, lead

    @property
    def shape(self):
        return torch.Size((*self._lead, self.cols))

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return "MicroscaledTensor(shape=%s, format=%s, device=%s)" % (tuple(self.shape), self.format, self.device)

    def block_scales(self):
        """``(..., ceil(cols / 32))`` scales as ``torch.float8_e8m0fnu`` (a view)."""
        return _host.block_scales(self.scales, self.cols, self._lead)

    def elements(self):
        """``(..., cols)`` element values before the scale, as ``torch.float8_e4m3fn``: a view for ``"mxfp8"``,
        unpacked for ``"mxfp4"`` (every e2m1 value is an e4m3 value)."""
        return _host.elements(self.codes, self.cols, self._lead, FORMATS[self.format])

    def dequantize(self, dtype=torch.float32):
        """The values ``element * scale`` (exact in fp32; rounded to nearest even in bfloat16 and float16)."""
        return _host.dequantize(self.codes, self.scales, self.cols, self._lead, FORMATS[self.format], dtype)


def _made(blocks, format):
    """The tensor of blocks that a call has just written."""
    q = MicroscaledTensor.__new__(MicroscaledTensor)
    q.codes, q.scales, q.rows, q.cols, q._lead = blocks
    q.format = format
    return q


def quantize(input, format="mxfp4"):
    """``(..., cols)`` float32 / bfloat16 / float16 -> :class:`MicroscaledTensor`."""
    return _made(_host.quantize(input, _format(format)), format)


def linear(input, weight, bias=None, activations="mxfp8", dtype=None, out=None):
    """``y = x W^T + b`` with both operands microscaled: ``weight`` a :class:`MicroscaledTensor` of ``(out, in)``,
    ``input`` either one of ``(..., in)`` or a plain tensor, which is quantised to ``activations`` on the way.

    Products are accumulated in fp32 and rounded once to ``dtype`` (default: the type of a plain input, float32 for a
    microscaled one).  8-bit activations take weights of either format, 4-bit activations 4-bit weights.  ``out``
    receives the result if given (contiguous, of the result's type and number of elements, over none of the operands)."""
    if not isinstance(weight, MicroscaledTensor) or len(weight._lead) != 1:
        raise RuntimeError("weight must be a MicroscaledTensor of (out_features, in_features)")
    if isinstance(input, MicroscaledTensor):
        return _host.linear(input.codes, input.scales, input._lead, input.cols, FORMATS[input.format], weight.codes,
                            weight.scales, weight.cols, FORMATS[weight.format], bias, dtype, out)
    return _host.linear(input, None, None, 0, _format(activations, "activations"), weight.codes, weight.scales,
                        weight.cols, FORMATS[weight.format], bias, dtype, out)


def rms_norm(input, weight=None, eps=1e-6, residual=None, noise=None, antithetic=False, output=None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, with ``h = input + residual``.

    ``weight`` is a float32 gain per column (ones if None).  ``residual`` has the input's shape and type; with it the
    call returns ``(y, h)``, ``h`` rounded to that type (``y`` is computed from the unrounded sum).  ``noise``
    ``(members, cols)`` float32 adds ``noise[d]`` to the gain of the rows ``r * members + d`` (its negative for the
    second half of the repeats with ``antithetic``).  ``output`` is None for a ``y`` of the input's type, or
    ``"mxfp8"`` / ``"mxfp4"`` for a :class:`MicroscaledTensor`.  Squares are summed in fp32: a row with magnitudes above
    1e19 has an infinite mean and is normalised to zeros, and magnitudes below 1e-19 lose bits in it, which an ``eps`` above
    1e-38 hides.  A value of ``y`` exactly between two codes takes the even one."""
    if output is None or output == getattr(input, "dtype", None):
        return _host.rms_norm(input, weight, eps, residual, noise, antithetic, 0)
    got = _host.rms_norm(input, weight, eps, residual, noise, antithetic, _format(output, "output"))
    return _made(got, output) if residual is None else (_made(got[0], output), got[1])


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
        bias = self.bias if self.bias is None or self.bias.dtype == torch.float32 else self.bias.float()
        return linear(input, self.weight, bias, self.activations, dtype)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s, format=%s, activations=%s" % (
            self.in_features, self.out_features, self.bias is not None, self.format, self.activations)
