"""Microscaled quantisation, RMS norm and product on the GPU against their 64-bit restatement.

Bounds.  Quantisation is exact arithmetic: bytes are compared for equality.  The norm's y differs from the 64-bit value
by at most DELTA = 24 * 2^-24 relative: at most 32 additions in any chain of the sum of squares (half of that reaches
the root), and one rounding each for x + residual, the sum / cols, + eps, the root, the gain and the product; a
quantised y must then be the code of some value within DELTA.  The product's terms are exact in fp32; the sum over K
adds K / 32 blocks, each summed with at most 8 roundings, so it is off by at most (K / 32 + 8) * 2^-23 * sum |x w|
(2^-23: an addition in the tensor pipe may truncate), then the bias and the result's type each round once.
"""
import numpy as np
import pytest
import torch

from oracle import microscaled_ref as O

pytestmark = pytest.mark.gpu

DELTA = 24 * 2.0 ** -24
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _ms():
    from nesgpu_b200 import microscaling
    return microscaling


def _f64(t):
    return t.detach().cpu().double().numpy()


def _inputs(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    x = x * torch.where(torch.rand(cols, generator=g) > 0.98, 16.0, 1.0) * scale
    return x.to(DTYPES[dtype]).cuda()


def _weight(ms, outs, cols, form, seed):
    """A random matrix in stored form and its values in float64."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(outs, cols, generator=g) / cols ** 0.5).double().numpy()
    codes, scales = O.quantize(w, form)
    packed, s = O.pack(codes, scales, form)
    return ms.MicroscaledTensor(torch.from_numpy(packed).cuda(), torch.from_numpy(s).cuda(), cols, form), O.values(codes, scales, form)


def _check_quantized(q, x64, form):
    codes, scales = O.quantize(x64, form)
    packed, s = O.pack(codes, scales, form)
    assert np.array_equal(q.scales.cpu().numpy(), s)
    assert np.array_equal(q.codes.cpu().numpy(), packed)


# ------------------------------------------------------------------------------------------------ quantisation

@pytest.mark.parametrize("form", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 128), (4, 129), (7, 200), (1, 4096), (33, 1000),
                                       (130, 257), (64, 2048), (1, 16385)])
def test_quantize(rows, cols, dtype, form):
    ms = _ms()
    x = _inputs(rows, cols, dtype, rows * 7 + cols)
    q = ms.quantize(x, form)
    assert tuple(q.shape) == (rows, cols) and q.format == form
    _check_quantized(q, _f64(x), form)
    codes, scales = O.quantize(_f64(x), form)
    assert np.array_equal(_f64(q.elements()), O.elements(codes, form))
    assert np.array_equal(q.block_scales().contiguous().view(torch.uint8).cpu().numpy(), scales)
    want = O.values(codes, scales, form)
    assert np.array_equal(_f64(q.dequantize()), want)
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(q.dequantize(t).cpu(), torch.from_numpy(want).float().to(t))


@pytest.mark.parametrize("form", ["mxfp4", "mxfp8"])
def test_quantize_special_blocks(form):
    """Zero blocks, subnormal and largest values, exact powers of two and their neighbours, ties, saturation, NaN, inf."""
    ms = _ms()
    one = np.float32(1)
    rows = [np.zeros(64), np.full(64, -0.0), np.full(64, 2.0 ** -149), np.full(64, 2.0 ** -126), np.full(64, 3.4e38)]
    rows += [np.full(64, v) for v in (1.0, 2.0, np.nextafter(one * 2, one), np.nextafter(one * 2, one * 3), 1.75, 1.9999)]
    ties = np.tile([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5], 8)
    rows += [ties, -ties, ties * 2.0 ** -130, ties * 2.0 ** 120, np.linspace(-512, 512, 64), np.arange(64) * 2.0 ** -11]
    x = np.stack(rows).astype(np.float32)
    bad = np.random.default_rng(0).standard_normal((4, 64)).astype(np.float32)
    bad[0, 3], bad[1, 40], bad[2, 0], bad[3, 63] = np.nan, np.inf, -np.inf, -np.nan
    x = np.concatenate([x, bad])
    q = ms.quantize(torch.from_numpy(x).cuda(), form)
    _check_quantized(q, x.astype(np.float64), form)
    codes, scales = O.quantize(x.astype(np.float64), form)
    assert np.array_equal(_f64(q.dequantize()), O.values(codes, scales, form), equal_nan=True)


def test_quantize_leading_dimensions_strides_and_alignment():
    ms = _ms()
    x = _inputs(60, 96, "bf16", 5)
    q = ms.quantize(x.view(3, 4, 5, 96))
    assert tuple(q.shape) == (3, 4, 5, 96) and tuple(q.elements().shape) == (3, 4, 5, 96)
    assert tuple(q.block_scales().shape) == (3, 4, 5, 3) and tuple(q.dequantize().shape) == (3, 4, 5, 96)
    _check_quantized(q, _f64(x), "mxfp4")
    wide = _inputs(9, 300, "fp32", 6)
    _check_quantized(ms.quantize(wide[:, 7:200], "mxfp8"), _f64(wide[:, 7:200]), "mxfp8")
    _check_quantized(ms.quantize(wide.t(), "mxfp8"), _f64(wide.t()), "mxfp8")
    flat = _inputs(1, 8 * 128 + 1, "fp16", 7).view(-1)
    off = flat[1:].view(8, 128)                       # rows start 2 bytes past a 16-byte boundary
    _check_quantized(ms.quantize(off, "mxfp4"), _f64(off), "mxfp4")
    row = ms.quantize(x[5], "mxfp8")                  # no leading dimension at all
    assert tuple(row.shape) == (96,) and tuple(row.elements().shape) == (96,) and tuple(row.block_scales().shape) == (3,)
    _check_quantized(row, _f64(x[5:6]), "mxfp8")
    empty = ms.quantize(torch.empty(0, 64, device="cuda"))
    assert tuple(empty.dequantize().shape) == (0, 64) and tuple(empty.elements().shape) == (0, 64)
    assert tuple(empty.block_scales().shape) == (0, 2)


def test_many_rows():
    """More rows than one pass of the grid covers."""
    ms = _ms()
    x = _inputs(70000, 40, "fp32", 8)
    q = ms.quantize(x, "mxfp8")
    _check_quantized(q, _f64(x), "mxfp8")
    codes, scales = O.quantize(_f64(x), "mxfp8")
    assert np.array_equal(_f64(q.dequantize()), O.values(codes, scales, "mxfp8"))


# -------------------------------------------------------------------------------------------------------- norm

def _check_norm(y, want, form, dtype):
    if form is None:
        half = torch.finfo(DTYPES[dtype]).eps / 2
        tiny = float(torch.finfo(DTYPES[dtype]).tiny) * half * 2          # spacing of the subnormals
        assert np.all(np.abs(_f64(y) - want) <= np.abs(want) * (DELTA + half * (1 + DELTA)) + tiny)
        return
    rows, cols = want.shape
    blocks = -(-cols // 32)
    p = np.zeros((rows, blocks * 32))
    p[:, :cols] = want
    largest = np.abs(p).reshape(rows, blocks, 32).max(axis=2)
    scales = y.scales.cpu().numpy()[:, :blocks]
    assert np.all(scales >= O.scale_codes(largest * (1 - DELTA), form)) and np.all(scales <= O.scale_codes(largest * (1 + DELTA), form))
    inverse = np.repeat(np.exp2(127.0 - scales), 32, axis=1)[:, :cols]
    lo = O.elements(O.element_codes(np.abs(want) * (1 - DELTA) * inverse, form), form)
    hi = O.elements(O.element_codes(np.abs(want) * (1 + DELTA) * inverse, form), form)
    got = _f64(y.elements())
    assert np.all(np.abs(got) >= lo) and np.all(np.abs(got) <= hi)
    assert np.all((got == 0) | (np.sign(got) == np.sign(want)))
    pad = y.codes.cpu().numpy().reshape(rows, -1)
    used = -(-cols // 2) if form == "mxfp4" else cols
    assert not pad[:, used:].any() and not y.scales.cpu().numpy()[:, blocks:].any()


@pytest.mark.parametrize("form", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols,members,with_residual,antithetic", [
    (1, 1, 0, False, False), (1, 33, 0, True, False), (6, 200, 3, True, True), (5, 256, 0, False, False), (9, 257, 9, False, True),
    (4, 512, 0, True, False), (12, 1000, 4, True, True), (3, 1024, 0, True, False), (2, 2048, 1, False, False), (1, 4096, 0, True, False),
    (3, 4097, 0, True, False), (2, 8192, 2, True, False), (2, 16384, 0, True, False), (3, 16389, 0, True, False), (2, 40000, 2, True, True),
    (9, 16383, 0, True, False), (3, 17400, 0, True, False), (4, 17411, 2, False, False), (700, 515, 7, True, True), (601, 1023, 0, True, False),
    (600, 1009, 0, True, False), (500, 250, 5, True, False), (420, 4099, 3, True, True), (300, 4350, 0, True, False), (640, 127, 0, True, False),
    (304, 256, 4, True, True), (310, 512, 0, False, False), (300, 1024, 3, True, False), (297, 2048, 0, True, False), (320, 4096, 5, True, True),
    (300, 8192, 0, True, False), (300, 1000, 6, False, True), (302, 2056, 2, True, False), (297, 5000, 0, True, False), (298, 17408, 0, False, False)])
def test_rms_norm(rows, cols, members, with_residual, antithetic, dtype, form):
    ms = _ms()
    x = _inputs(rows, cols, dtype, rows + cols)
    res = _inputs(rows, cols, dtype, rows + cols + 1, 0.5) if with_residual else None
    g = torch.Generator().manual_seed(cols)
    gain = (1 + 0.3 * torch.randn(cols, generator=g)).cuda()
    noise = (0.05 * torch.randn(members, cols, generator=g)).cuda() if members else None
    got = ms.rms_norm(x, gain, 1e-5, res, noise, antithetic, form)
    y, h = got if with_residual else (got, None)
    eps = float(np.float32(1e-5))
    want, h64 = O.rms_norm(_f64(x), _f64(gain), eps, None if res is None else _f64(res), None if noise is None else _f64(noise), antithetic)
    if h is not None:
        assert h.dtype == x.dtype and torch.equal(h, (x.float() + res.float()).to(x.dtype))
    # gain + noise rounds relative to their sum, which the bound on y counts; its operands may cancel
    _check_norm(y, want, form, dtype)


def test_rms_norm_defaults_and_shapes():
    ms = _ms()
    x = _inputs(24, 48, "bf16", 3)
    y = ms.rms_norm(x.view(2, 3, 4, 48))
    assert tuple(y.shape) == (2, 3, 4, 48) and y.dtype == torch.bfloat16
    want, _ = O.rms_norm(_f64(x), None, float(np.float32(1e-6)))
    _check_norm(y.view(24, 48), want, None, "bf16")
    assert torch.equal(ms.rms_norm(x[3]), ms.rms_norm(x)[3])
    y, h = ms.rms_norm(x.view(4, 6, 48), residual=x.view(4, 6, 48), output="mxfp8")
    assert tuple(y.shape) == (4, 6, 48) and tuple(h.shape) == (4, 6, 48)
    strided = _inputs(10, 100, "fp32", 4)[:, 3:60]
    want, _ = O.rms_norm(_f64(strided), None, float(np.float32(1e-6)))
    _check_norm(ms.rms_norm(strided), want, None, "fp32")
    assert ms.rms_norm(torch.empty(0, 8, device="cuda")).shape == (0, 8)
    flat = _inputs(1, 8 * 128 + 1, "bf16", 7).view(-1)
    off = flat[1:].view(8, 128)                       # rows start 2 bytes past a 16-byte boundary
    want, _ = O.rms_norm(_f64(off), _f64(flat[1:129].float()), float(np.float32(1e-6)))
    _check_norm(ms.rms_norm(off, flat.float()[1:129]), want, None, "bf16")


@pytest.mark.parametrize("form", [None, "mxfp8", "mxfp4"])
def test_rms_norm_special_rows(form):
    """A zero row is zero; a NaN or an infinity stays within its row; huge rows overflow to zero as the formula does in fp32."""
    ms = _ms()
    x = _inputs(6, 96, "fp32", 9)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 70] = float("inf")
    x[4] = x[4] * 1e-30
    y = ms.rms_norm(x, output=form)
    v = _f64(y if form is None else y.dequantize())
    assert not v[1].any()
    assert np.isnan(v[2]).all()
    assert np.isnan(v[3, 70]) and not np.isfinite(v[3, 64:96]).all() and not v[3, :64].any()
    keep = [0, 1, 4, 5]
    want, _ = O.rms_norm(_f64(x)[keep], None, float(np.float32(1e-6)))
    sub = ms.rms_norm(x[keep], output=form)
    _check_norm(sub, want, form, "fp32")


def test_rms_norm_pad_columns_stay_zero_when_the_root_is_infinite():
    ms = _ms()
    y = ms.rms_norm(torch.zeros(2, 40, device="cuda"), eps=0.0, output="mxfp8")       # 0 * inf = NaN in every column
    assert np.isnan(_f64(y.dequantize())).all()
    assert not y.codes[:, 40:].any() and not y.scales[:, 2:].any()


# ----------------------------------------------------------------------------------------------------- product

def _check_linear(y, x64, w64, bias, dtype):
    want, absolute = O.linear(x64, w64, None if bias is None else _f64(bias))
    K = x64.shape[1]
    half = torch.finfo(dtype).eps / 2
    bound = (K / 32 + 8) * 2.0 ** -23 * absolute
    bound = bound + 2.0 ** -24 * (np.abs(want) + bound) + half * (np.abs(want) + 2 * bound) + 2.0 ** -25 * torch.finfo(dtype).tiny
    assert y.dtype == dtype and tuple(y.shape) == want.shape
    err = np.abs(_f64(y) - want)
    assert np.all(err <= bound), "worst %g of its bound" % np.nanmax(err / bound)


PAIRS = [("mxfp4", "mxfp4"), ("mxfp8", "mxfp4"), ("mxfp8", "mxfp8")]
SIZES = [(1, 1, 1), (1, 128, 64), (1, 4096, 300), (2, 33, 5), (3, 200, 129), (8, 512, 128), (9, 1024, 257), (15, 96, 40), (16, 640, 1000),
         (17, 128, 128), (24, 2048, 384), (31, 65, 77), (33, 1000, 130), (64, 384, 256), (65, 256, 513), (100, 1536, 100), (128, 128, 128),
         (129, 160, 129), (200, 2049, 70), (256, 512, 256), (300, 1000, 513), (513, 1024, 1030)]


@pytest.mark.parametrize("activations,weights", PAIRS)
@pytest.mark.parametrize("rows,cols,outs", SIZES)
def test_linear(rows, cols, outs, activations, weights):
    ms = _ms()
    for dtype in ("fp32", "bf16"):
        x = _inputs(rows, cols, dtype, rows * 3 + cols)
        w, w64 = _weight(ms, outs, cols, weights, outs)
        bias = torch.randn(outs, generator=torch.Generator().manual_seed(1)).cuda()
        codes, scales = O.quantize(_f64(x), activations)
        x64 = O.values(codes, scales, activations)
        _check_linear(ms.linear(x, w, bias, activations), x64, w64, bias, DTYPES[dtype])
        y = ms.linear(ms.quantize(x, activations), w)
        _check_linear(y, x64, w64, None, torch.float32)


@pytest.mark.parametrize("activations,weights", PAIRS)
@pytest.mark.parametrize("rows,cols,outs", [(2100, 128, 5000), (1300, 1160, 7000), (4500, 700, 2305)])
def test_linear_more_tiles_than_processors(rows, cols, outs, activations, weights):
    test_linear(rows, cols, outs, activations, weights)


@pytest.mark.parametrize("activations,weights", PAIRS)
@pytest.mark.parametrize("rows", [1, 16, 40, 150])
def test_linear_special_scales(rows, activations, weights):
    """A NaN block poisons its own row or column only; scales at both ends of the range meet without overflow."""
    ms = _ms()
    x = _inputs(rows, 320, "fp32", 2)
    x[0, 33] = float("nan")
    w, w64 = _weight(ms, 70, 320, weights, 3)
    w.scales[5, 2] = 255
    y = _f64(ms.linear(x, w, None, activations))
    assert np.isnan(y[0]).all() and np.isnan(y[:, 5]).all()
    ok = np.ones(70, bool)
    ok[5] = False
    assert np.isfinite(y[1:][:, ok]).all()
    tiny, huge = _inputs(rows, 320, "fp32", 4) * 2.0 ** -100, None
    w, w64 = _weight(ms, 70, 320, weights, 3)
    w.scales.add_(90)                                       # 2^90 times the values (pad scales change: their codes are zero)
    codes, scales = O.quantize(_f64(tiny), activations)
    _check_linear(ms.linear(tiny, w, None, activations), O.values(codes, scales, activations), w64 * 2.0 ** 90, None, torch.float32)


def test_linear_types_shapes_and_out():
    ms = _ms()
    w, w64 = _weight(ms, 48, 64, "mxfp4", 0)
    x = _inputs(12, 64, "fp16", 1)
    codes, scales = O.quantize(_f64(x), "mxfp8")
    x64 = O.values(codes, scales, "mxfp8")
    assert torch.equal(ms.linear(x[3], w), ms.linear(x[3:4], w)[0]) and ms.linear(ms.quantize(x[3]), w).shape == (48,)
    y = ms.linear(x.view(3, 4, 64), w)
    assert tuple(y.shape) == (3, 4, 48) and y.dtype == torch.float16
    _check_linear(y.view(12, 48), x64, w64, None, torch.float16)
    _check_linear(ms.linear(x, w, dtype=torch.float32), x64, w64, None, torch.float32)
    out = torch.full((12, 48), 7.0, device="cuda", dtype=torch.bfloat16)
    assert ms.linear(x, w, out=out) is out
    _check_linear(out, x64, w64, None, torch.bfloat16)
    assert tuple(ms.linear(torch.empty(0, 64, device="cuda"), w).shape) == (0, 48)
    assert tuple(ms.linear(ms.quantize(torch.empty(0, 64, device="cuda")), w).shape) == (0, 48)


def test_rows_do_not_depend_on_their_neighbours():
    """A token's result is the same bits in any batch of one kernel's range, and outputs behind the last row stay as they were."""
    ms = _ms()
    w, _ = _weight(ms, 200, 512, "mxfp4", 0)
    x = _inputs(300, 512, "bf16", 1)
    buf = torch.full((301, 200), 3.0, device="cuda", dtype=torch.bfloat16)
    ms.linear(x, w, activations="mxfp4", out=buf[:300])
    assert (buf[300] == 3).all()
    again = ms.linear(x, w, activations="mxfp4")
    assert torch.equal(buf[:300], again)
    w, _ = _weight(ms, 4104, 512, "mxfp4", 0)                # and through boxes that are cut off at the edges
    x = _inputs(1100, 512, "bf16", 1)
    for dtype in (torch.bfloat16, torch.float32):
        buf = torch.full((1101, 4104), 3.0, device="cuda", dtype=dtype)
        ms.linear(x, w, out=buf[:1100])
        assert (buf[1100] == 3).all() and torch.equal(buf[:1100], ms.linear(x, w, dtype=dtype))


# ---------------------------------------------------------------------------------------------------- refusals

def test_refusals():
    ms = _ms()
    x = torch.zeros(4, 64, device="cuda")
    q = ms.quantize(x)
    with pytest.raises(NotImplementedError, match="float64"):
        ms.quantize(x.double())
    with pytest.raises(RuntimeError, match="column"):
        ms.quantize(x[:, :0])
    with pytest.raises(RuntimeError, match="last dimension"):
        ms.linear(x[:, :32], q)
    with pytest.raises(NotImplementedError, match="formats"):
        ms.linear(x, ms.quantize(x, "mxfp8"), activations="mxfp4")
    with pytest.raises(RuntimeError, match="bias"):
        ms.linear(x, q, torch.zeros(5, device="cuda"))
    with pytest.raises(RuntimeError, match="out must"):
        ms.linear(x, q, out=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(RuntimeError, match="codes and scales"):
        ms.MicroscaledTensor(q.codes, q.scales, 200)
    with pytest.raises(RuntimeError, match="leading"):
        ms.MicroscaledTensor(q.codes, q.scales, 64, shape=(3,))
    with pytest.raises(RuntimeError, match="residual"):
        ms.rms_norm(x, residual=x[:2])
    with pytest.raises(NotImplementedError, match="residual"):
        ms.rms_norm(x, residual=x.half())
    with pytest.raises(RuntimeError, match="multiple of directions"):
        ms.rms_norm(x, noise=torch.zeros(3, 64, device="cuda"))
    with pytest.raises(NotImplementedError, match="output"):
        ms.rms_norm(x, output="mxfp6")
    with pytest.raises(RuntimeError, match="eps"):
        ms.rms_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ms.linear(x, q, torch.zeros(4))
    with pytest.raises(RuntimeError, match="weight must"):
        ms.rms_norm(x, torch.ones(32, device="cuda"))
    with pytest.raises(NotImplementedError, match="bfloat16"):
        ms.rms_norm(x, torch.ones(64, device="cuda").bfloat16())
    with pytest.raises(NotImplementedError, match="int32"):
        ms.linear(x, q, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ms.linear([1.0], q)


def test_refusals_of_blocks_changed_since():
    """The object's tensors can be replaced; what no longer fits together is refused where it is used."""
    ms = _ms()
    x = torch.ones(4, 256, device="cuda")
    w = ms.quantize(torch.ones(8, 256, device="cuda"))
    for form in ("mxfp4", "mxfp8"):
        good = ms.quantize(x, form)
        more, narrow = ms.quantize(torch.ones(6, 256, device="cuda"), form), ms.quantize(x[:, :128], form)
        for codes, scales in ((more.codes, more.scales), (more.codes, good.scales), (narrow.codes, good.scales), (good.codes, narrow.scales),
                              (good.codes.int(), good.scales), (good.codes, good.scales.t().contiguous().t())):
            q = ms.quantize(x, form)
            q.codes, q.scales = codes, scales
            for call in (q.dequantize, lambda: ms.linear(q, w)):
                with pytest.raises(RuntimeError, match="microscaled tensor must|leading"):
                    call()
            if codes is not good.codes:
                with pytest.raises(RuntimeError, match="microscaled tensor must|leading"):
                    q.elements()
        w2 = ms.quantize(torch.ones(8, 256, device="cuda"))
        w2.scales = good.scales
        with pytest.raises(RuntimeError, match="microscaled tensor must"):
            ms.linear(x, w2)


@pytest.mark.parametrize("rows", [1, 40])
def test_results_over_inputs_are_refused(rows):
    ms = _ms()
    C = pytest.importorskip("nesgpu_b200._cabi")
    x = torch.ones(rows, 256, device="cuda")
    w = ms.quantize(torch.ones(256, 256, device="cuda"))
    with pytest.raises(C.NesError, match="overlap"):
        ms.linear(x, w, out=x)
    both = torch.ones(2 * rows, 256, device="cuda")
    y = ms.linear(both[:rows], w, out=both[rows:])              # next to one another
    assert torch.equal(y, torch.full_like(y, 256.0))
