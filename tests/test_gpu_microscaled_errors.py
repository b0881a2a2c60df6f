"""Errors of the microscaled calls on the GPU: each is the exception that PyTorch or Python raised, and nothing is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_failed_allocation_is_out_of_memory():
    """2^42 elements at least, which no card holds: code that catches the error to make its batch smaller goes on as with
    the other layers."""
    from nesgpu_b200 import microscaling as ms
    large = torch.zeros(1, 64, device="cuda").expand(1 << 36, 64)
    with pytest.raises(torch.OutOfMemoryError):
        ms.quantize(large)
    with pytest.raises(torch.OutOfMemoryError):
        ms.rms_norm(large)
    many = ms.quantize(torch.ones(1 << 21, 1, device="cuda"))
    x = torch.ones(1 << 21, 1, device="cuda", dtype=torch.bfloat16)
    for activations in (x, ms.quantize(x, "mxfp8")):
        with pytest.raises(torch.OutOfMemoryError):
            ms.linear(activations, many)
    y = ms.linear(x[:3], many)                            # and the next call works
    assert y.shape == (3, 1 << 21) and bool((y == 1).all())


def test_an_argument_without_a_truth_value_is_refused():
    from nesgpu_b200 import microscaling as ms
    x = torch.ones(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="ambiguous"):
        ms.rms_norm(x, noise=torch.zeros(2, 64, device="cuda"), antithetic=torch.ones(2))

    class Without:
        def __bool__(self):
            raise KeyError("no truth value")

    with pytest.raises(KeyError, match="no truth value"):
        ms.rms_norm(x, antithetic=Without())
    assert bool((ms.rms_norm(x, eps=0.0) == 1).all())
