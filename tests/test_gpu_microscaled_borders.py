"""Quantised norm outputs whose exact values lie on a border between two codes, or on a power of two that decides a block's scale.

Rows hold whole numbers with mean(h^2) = root^2 exactly and gains that are multiples of 2^-10, so y = h * gain / root is known exactly:
the product in 64 bits is exact and the quotient is rounded to 64 bits once, which leaves every border (a number of few bits)
what it is.  A quotient n / (15 * 2^10) that is no border b * 2^-j (b of five bits) differs from it by 2^-20 of its size at least,
so the codes must be equal and no tolerance is taken.  eps is 0, or so small beside the mean that it vanishes in 64 bits.
"""
import numpy as np
import pytest
import torch

from oracle import microscaled_ref as O

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# eight whole numbers whose squares add up to 8 * root^2
PATTERNS = {3: [6, 4, 4, 2, 0, 0, 0, 0], 4: [5, 9, 3, 3, 2, 0, 0, 0], 5: [12, 6, 4, 2, 0, 0, 0, 0], 15: [30, 20, 16, 12, 8, 6, 0, 0]}
SIZES = [(1, 40), (9, 257), (5, 256), (2, 1000), (4, 1024), (600, 512), (300, 2048), (500, 4096), (3, 4097), (299, 4099),
         (2, 17600), (2, 17411)]


def _rows(rows, cols, seed):
    """Whole numbers (rows, cols) and the root of every row's mean square."""
    rng = np.random.default_rng(seed)
    h, root = np.empty((rows, cols)), rng.choice(list(PATTERNS), rows).astype(np.float64)
    for r in range(rows):
        row = np.full(cols, root[r])
        row[:cols // 8 * 8] = np.tile(PATTERNS[int(root[r])], cols // 8)
        h[r] = rng.permutation(row) * rng.choice([-1, 1], cols) + 0.0          # no negative zeros
    assert np.array_equal((h * h).sum(axis=1), cols * root * root)
    return h, root[:, None]


def _gains(shape, seed):
    """Mostly gains of few bits, which put many y on borders."""
    rng = np.random.default_rng(seed)
    few, many = rng.integers(1, 33, shape) / 16.0, rng.integers(512, 2049, shape) / 1024.0
    return np.where(rng.random(shape) < 0.8, few, many)


def _on_borders(y, form):
    """How many values lie exactly between two codes of their block."""
    codes, scales = O.quantize(y, form)
    v = np.abs(y) * np.exp2(127.0 - np.repeat(scales, 32, axis=1)[:, :y.shape[1]])
    table = O.MAGNITUDES if form == "mxfp4" else O.e4m3_values()[:127]
    return int(np.isin(v, (table[1:] + table[:-1]) / 2).sum())


def test_rows_lie_on_borders():
    """What the tests below are made of, without a GPU: they hold ties in both formats."""
    ties = {"mxfp4": 0, "mxfp8": 0}
    for rows, cols in SIZES[:5]:
        h, root = _rows(rows, cols, rows)
        y = h * _gains(cols, cols) / root
        for form in ties:
            ties[form] += _on_borders(y, form)
    assert ties["mxfp4"] >= 100 and ties["mxfp8"] >= 20, ties
    y = np.tile(np.array(PATTERNS[4], np.float64), 4)[None] / 4          # 1.25 of a largest 2.25: 2.5 goes to the even 2, not to 3
    assert O.elements(O.quantize(y, "mxfp4")[0], "mxfp4")[0, 0] == 2


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_rms_norm_on_borders(rows, cols, dtype, form):
    from nesgpu_b200 import microscaling as ms
    h, root = _rows(rows, cols, rows + cols)
    gain = _gains(cols, cols)
    members = 3 if rows % 3 == 0 else 1
    noise = _gains((members, cols), rows)
    r = np.arange(rows) // members
    sign = np.where(r >= (rows // members + 1) // 2, -1.0, 1.0)[:, None]
    part = np.random.default_rng(2).integers(-8, 9, h.shape)
    scale = np.exp2(np.random.default_rng(3).integers(-9, 10 if dtype == "fp16" else 30, (rows, 1)))     # the same y
    t = lambda a, kind=torch.float32: torch.from_numpy(a).to(kind).cuda()

    def check(q, want):
        codes, scales = O.quantize(want, form)
        packed, s = O.pack(codes, scales, form)
        assert np.array_equal(q.scales.cpu().numpy(), s)
        assert np.array_equal(q.elements().cpu().double().numpy(), O.elements(codes, form))        # a zero of either sign
        used = -(-cols // 2) if form == "mxfp4" else cols
        assert not q.codes[:, used:].any()

    x = t(h, DTYPES[dtype])
    check(ms.rms_norm(x, eps=0.0, output=form), h / root)
    check(ms.rms_norm(x, t(gain), eps=0.0, output=form), h * gain / root)
    check(ms.rms_norm(x, t(gain), eps=1e-24, output=form), h * gain / root)                # 2^-79 beside a mean of at least 9
    check(ms.rms_norm(t(h * scale, DTYPES[dtype]), t(gain), eps=0.0, output=form), h * gain / root)
    q, got = ms.rms_norm(t(h - part, DTYPES[dtype]), t(gain), 0.0, t(part.astype(np.float64), DTYPES[dtype]), output=form)
    assert np.array_equal(got.cpu().double().numpy(), h)
    check(q, h * gain / root)
    # row r * members + d; ties of a sum that cancels to few bits
    g = gain + sign * noise[np.arange(rows) % members]
    check(ms.rms_norm(x, t(gain), 0.0, noise=t(noise), antithetic=True, output=form), h * g / root)
