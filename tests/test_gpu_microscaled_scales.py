"""Block scales at the ends of their range in the product."""
import numpy as np
import pytest
import torch

from oracle import microscaled_ref as O
from test_gpu_microscaled import PAIRS, _check_linear

pytestmark = pytest.mark.gpu


def _operand(ms, rows, cols, form, codes_of_scale, seed):
    """Random elements whose blocks have the given scale codes, as a tensor and as values in 64 bits."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16 if form == "mxfp4" else 0x50, (rows, cols)).astype(np.uint8)
    if form == "mxfp8":
        codes |= (rng.integers(0, 2, (rows, cols)) << 7).astype(np.uint8)
    scales = np.broadcast_to(codes_of_scale, (rows, -(-cols // 32))).astype(np.uint8)
    packed, s = O.pack(codes, scales, form)
    return ms.MicroscaledTensor(torch.from_numpy(packed).cuda(), torch.from_numpy(s).cuda(), cols, form), O.values(codes, scales, form)


# single CTAs of 16, 32, 64 and 128 tokens, K in one part and in several, CTA pairs
@pytest.mark.parametrize("activations,weights", PAIRS)
@pytest.mark.parametrize("rows,cols,outs", [(3, 320, 70), (20, 2048, 130), (50, 4096, 128), (130, 320, 257), (100, 4096, 100), (1300, 256, 7000)])
def test_smallest_scales_meet_the_largest(rows, cols, outs, activations, weights):
    """2^-127 times 2^127, in both orders and side by side in one row: finite products of ordinary size."""
    from nesgpu_b200 import microscaling as ms
    blocks = cols // 32
    both = np.where(np.arange(blocks) % 2 == 0, 0, 254)
    for x_scales, w_scales in ((np.zeros(blocks), np.full(blocks, 254)), (np.full(blocks, 254), np.zeros(blocks)), (both, 254 - both)):
        x, x64 = _operand(ms, rows, cols, activations, x_scales, 1)
        w, w64 = _operand(ms, outs, cols, weights, w_scales, 2)
        _check_linear(ms.linear(x, w), x64, w64, None, torch.float32)
        _check_linear(ms.linear(x, w, dtype=torch.bfloat16), x64, w64, None, torch.bfloat16)


@pytest.mark.parametrize("activations,weights", PAIRS)
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_scales_beyond_the_range_of_fp32_together(rows, activations, weights):
    """Both smallest: every product is below the smallest fp32 and the result is zero.  Both largest: no sum is finite."""
    from nesgpu_b200 import microscaling as ms
    for code in (0, 254):
        scales = np.full(10, code)
        x, x64 = _operand(ms, rows, 320, activations, scales, 3)
        w, w64 = _operand(ms, 70, 320, weights, scales, 4)
        y = ms.linear(x, w).cpu().double().numpy()
        want, absolute = O.linear(x64, w64, None)
        if code == 0:
            assert np.abs(want).max() < 2.0 ** -230 and not y.any()
        else:
            sure = np.abs(want) > absolute * 2.0 ** -20                # 2^254 and more, unless elements cancel
            assert not np.isfinite(y[sure]).any()
