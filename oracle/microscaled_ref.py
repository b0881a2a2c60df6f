"""Microscaled quantisation, RMS norm and product restated in 64 bits on the CPU (numpy), from their definitions."""
import numpy as np

BLOCK = 32
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """The 256 values of an e4m3 byte (no infinities; 0x7f and 0xff are NaN)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[c] = np.nan if (c & 127) == 127 else (-v if s else v)
    return out


_E4M3 = e4m3_values()


def pitches(cols, form):
    groups = -(-cols // 128)
    return groups * (64 if form == "mxfp4" else 128), groups * 4


def _nearest(v, table):
    """Index of the table entry (ascending, not negative) nearest to v >= 0; ties to the even index; saturated."""
    hi = np.clip(np.searchsorted(table, v), 0, len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = table[hi] - v, v - table[lo]
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    return np.where(v >= table[-1], len(table) - 1, np.where(take_hi, hi, lo))


def element_codes(scaled, form):
    """Code of every scaled value (float64), without packing."""
    table = MAGNITUDES if form == "mxfp4" else _E4M3[:127]
    code = _nearest(np.abs(scaled), table)
    return (code | (np.signbit(scaled) << (3 if form == "mxfp4" else 7))).astype(np.uint8)


def scale_codes(largest, form):
    """Code of the block scale from the block's largest magnitude (NaN or inf: 255)."""
    emax = 2 if form == "mxfp4" else 8
    bad = ~np.isfinite(largest)
    _, e = np.frexp(np.where(bad | (largest == 0), 1.0, largest))
    code = np.clip(e - 1 - emax + 127, 0, 254)
    return np.where(bad, 255, np.where(largest == 0, 0, code)).astype(np.uint8)


def quantize(x, form):
    """x (rows, cols) float64 -> (element codes (rows, cols), scale codes (rows, blocks))."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    p = np.zeros((rows, blocks * BLOCK))
    p[:, :cols] = x
    p = p.reshape(rows, blocks, BLOCK)
    with np.errstate(invalid="ignore"):
        largest = np.abs(p).max(axis=2)               # NaN if the block holds one
    scales = scale_codes(largest, form)
    bad = scales == 255
    scaled = np.where(bad[..., None], 0.0, np.where(bad[..., None], 0.0, p) * np.exp2(127.0 - np.where(bad, 127, scales))[..., None])
    return element_codes(scaled, form).reshape(rows, -1)[:, :cols], scales


def pack(codes, scales, form):
    """Stored form: rows padded to groups of 128 elements, two 4-bit codes to a byte."""
    rows, cols = codes.shape
    pitch, spitch = pitches(cols, form)
    full = np.zeros((rows, pitch * (2 if form == "mxfp4" else 1)), dtype=np.uint8)
    full[:, :cols] = codes
    s = np.zeros((rows, spitch), dtype=np.uint8)
    s[:, :scales.shape[1]] = scales
    if form == "mxfp4":
        full = full[:, 0::2] | (full[:, 1::2] << 4)
    return full, s


def elements(codes, form):
    """Element values of codes."""
    if form == "mxfp4":
        v = MAGNITUDES[codes & 7]
        return np.where(codes & 8, -v, v)
    return _E4M3[codes]


def values(codes, scales, form):
    """element * scale, float64; NaN in blocks of scale 255."""
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return elements(codes, form) * np.repeat(s, BLOCK, axis=1)[:, :codes.shape[1]]


def rms_norm(x, gain, eps, residual=None, noise=None, antithetic=False):
    """(y, h) in float64."""
    h = x if residual is None else x + residual
    rows = h.shape[0]
    g = np.ones(h.shape[1]) if gain is None else gain
    g = np.broadcast_to(g, h.shape)
    if noise is not None:
        D = noise.shape[0]
        r, d = np.arange(rows) // D, np.arange(rows) % D
        sign = np.where(antithetic & (r >= (rows // D + 1) // 2), -1.0, 1.0)
        g = g + sign[:, None] * noise[d]
    return h / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps) * g, h


def linear(x, w, bias):
    """x, w: float64 values; returns (y, sum of |products|), the second for error bounds."""
    y = x @ w.T
    if bias is not None:
        y = y + bias
    return y, np.abs(x) @ np.abs(w).T
