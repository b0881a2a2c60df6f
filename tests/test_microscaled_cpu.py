"""Microscaled operators without a GPU: the oracle against torch's own 8-bit types, refusals, host-side layer logic."""
import numpy as np
import pytest
import torch

from oracle import microscaled_ref as O


def test_oracle_e4m3_table_is_torchs():
    got = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    want = O.e4m3_values()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


def test_oracle_e4m3_rounding_is_torchs():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 9, (20000,), generator=g).float()),
                   torch.arange(-4480, 4481) / 10, torch.arange(-600, 601) * 2.0 ** -10]).clamp(-448, 448)
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.element_codes(x.double().numpy(), "mxfp8"), want)


def test_oracle_e2m1_ties_go_to_the_even_code():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9])
    assert O.elements(O.element_codes(ties, "mxfp4"), "mxfp4").tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 6]
    assert O.element_codes(-ties[:1], "mxfp4").tolist() == [8]


@pytest.mark.parametrize("form,emax", [("mxfp4", 2), ("mxfp8", 8)])
def test_oracle_scale_codes(form, emax):
    largest = np.array([0.0, 1.0, 1.999, 2.0, 2.0 ** -149, 2.0 ** 127 * 1.5, np.inf, np.nan])
    assert O.scale_codes(largest, form).tolist() == [0, 127 - emax, 127 - emax, 128 - emax, 0, 254 - emax, 255, 255]


def test_refusals():
    from nesgpu_b200 import microscaling as ms
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ms.quantize(x)
    with pytest.raises(NotImplementedError, match="format"):
        ms.quantize(x, "mxfp6")
    with pytest.raises(RuntimeError, match="CUDA"):
        ms.rms_norm(x)
    with pytest.raises(RuntimeError, match="MicroscaledTensor"):
        ms.linear(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ms.MicroscaledTensor(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), 64)
    with pytest.raises(NotImplementedError, match="4-bit weights"):
        ms.MicroscaledLinear(64, 64, format="mxfp8", activations="mxfp4")


def test_c_entry_refusals():
    """Bad extents, formats, pointers and workspaces come back as statuses; nothing is launched."""
    from nesgpu_b200 import _cabi
    L = _cabi.lib
    p = 4096                                        # stands for a device pointer; no call gets as far as using it
    assert L.nes_mx_quantize(p, 0, p, p, -1, 64, 4, None) == -1
    assert L.nes_mx_quantize(p, 0, p, p, 2, 64, 5, None) == -2
    assert L.nes_mx_quantize(p, 3, p, p, 2, 64, 4, None) == -2
    assert L.nes_mx_quantize(None, 0, p, p, 2, 64, 4, None) == -1
    assert L.nes_mx_quantize(p, 0, p + 8, p, 2, 64, 4, None) == -1
    assert L.nes_mx_quantize(None, 0, None, None, 0, 64, 4, None) == 0
    assert L.nes_mx_dequantize(p, p, None, 0, 2, 64, 8, None) == -1
    assert L.nes_mx_elements(p, None, 2, 64, None) == -1
    assert L.nes_rms_norm_fwd(p, p, None, p, None, p, None, 2, 64, 0, 0, 0, 0, 1e-6, None) == -1      # residual, no output
    assert L.nes_rms_norm_fwd(p, None, None, p, None, p, None, 2, 64, 0, 0, 0, 8, 1e-6, None) == -1   # no scales
    assert L.nes_rms_norm_fwd(p, None, None, p, p, p, None, 3, 64, 2, 0, 0, 0, 1e-6, None) == -1      # 3 rows, 2 members
    assert L.nes_mx_linear_fwd(p, p, 0, 4, p, p, 8, None, p, 0, 2, 64, 64, None, 0, None) == -2       # 4-bit x, 8-bit w
    assert L.nes_mx_linear_fwd(p, p, 0, 4, p, p, 4, None, p, 0, 2, 64, 0, None, 0, None) == -1        # no columns
    assert L.nes_mx_linear_fwd(p, p, 0, 4, p + 4, p, 4, None, p, 0, 2, 64, 64, None, 0, None) == -1   # misaligned
    need = L.nes_mx_linear_fwd_scratch_bytes(200, 64, 64, 8)
    assert need >= 200 * (128 + 4)
    assert L.nes_mx_linear_fwd(p, None, 0, 8, p, p, 4, None, p, 0, 200, 64, 64, p, need - 1, None) == -5
    assert L.nes_mx_linear_fwd(p, None, 7, 8, p, p, 4, None, p, 0, 200, 64, 64, p, need, None) == -2
    assert L.nes_mx_linear_fwd(None, None, 0, 8, None, None, 4, None, None, 0, 0, 64, 64, None, 0, None) == 0


def test_norm_layer_state_follows_the_other_layers():
    from nesgpu_b200 import base
    import modules.base as mb
    assert mb.PerturbedRMSNorm is base.PerturbedRMSNorm
    layer = base.PerturbedRMSNorm(48, 6)
    assert layer.weight_noise is None and layer.bias is None and not layer.perturbed_flag
    layer.allocate_memory()
    assert layer.weight_noise.shape == (6, 48)
    layer.free_memory()
    assert layer.weight_noise is None
    assert [n for n, _ in layer.named_parameters()] == ["weight"]
    with pytest.raises(NotImplementedError, match="last dimension"):
        base.PerturbedRMSNorm((4, 8), 2)
    with pytest.raises(NotImplementedError, match="direct"):
        base.PerturbedRMSNorm(8, 2, options={"direct": True})
    pm = base.PerturbedModel(torch.nn.Sequential(layer, base.PerturbedLinear(48, 5, 6, options={"tc": "mxfp4"})), 6)
    assert len(pm.perturbed_layers) == 2


def test_outputs_over_inputs_are_refused():
    """Before anything reaches a device, so the addresses are made up."""
    from nesgpu_b200 import _cabi as C
    f32, mx4, mx8 = 0, 4, 8
    a, b, c, d, e = (n << 40 for n in range(1, 6))
    over = a + 4 * 128 * 4 - 16                      # the last bytes of a (4, 128) fp32 matrix at a
    calls = [("nes_mx_quantize", (a, f32, over, b, 4, 128, mx8, 0)),
             ("nes_mx_quantize", (a, f32, b, over, 4, 128, mx8, 0)),
             ("nes_mx_dequantize", (a, b, a + 4 * 128 - 16, f32, 4, 128, mx8, 0)),
             ("nes_mx_dequantize", (a, b, b, f32, 4, 128, mx8, 0)),
             ("nes_mx_elements", (a, a + 4 * 64 - 16, 4, 128, 0)),
             ("nes_mx_linear_fwd", (a, None, f32, mx8, b, c, mx4, None, over, f32, 4, 64, 128, None, 0, 0)),
             ("nes_mx_linear_fwd", (a, d, f32, mx8, b, c, mx4, None, d, f32, 4, 64, 128, None, 0, 0)),
             ("nes_mx_linear_fwd", (a, d, f32, mx8, b, c, mx4, e, e + 64 * 4 - 4, f32, 4, 64, 128, None, 0, 0)),
             ("nes_rms_norm_fwd", (a, None, None, None, None, a, None, 4, 128, 0, 0, f32, 0, 1e-6, 0)),
             ("nes_rms_norm_fwd", (a, b, b, None, None, c, None, 4, 128, 0, 0, f32, 0, 1e-6, 0)),
             ("nes_rms_norm_fwd", (a, None, None, b, c, c, d, 4, 128, 2, 0, f32, mx8, 1e-6, 0))]
    for name, args in calls:
        with pytest.raises(C.NesError, match="overlap"):
            C.call(name, *args)


@pytest.mark.parametrize("mode", ["mxfp4", "mxfp8", "mxfp8_mxfp4"])
def test_direct_storage_has_no_microscaled_mode(mode):
    """The population forward would run in fp32, the unperturbed one of the same layer in blocks."""
    from nesgpu_b200 import base
    with pytest.raises(NotImplementedError, match="direct storage"):
        base.PerturbedLinear(32, 8, 2, options={"direct": True, "tc": mode})
    layer = base.PerturbedLinear(32, 8, 2, options={"direct": True})
    layer.options["tc"] = mode
    for population in (False, True):
        layer.perturbed_flag = population
        with pytest.raises(NotImplementedError, match="direct storage"):
            layer(torch.zeros(4, 32))
    assert base.PerturbedLinear(32, 8, 2, options={"direct": True, "tc": "tf32"}).options["direct"]


def test_the_layers_do_without_the_extension_module():
    """It is tied to one PyTorch; where it does not load, the microscaled calls say so and everything else works."""
    import subprocess
    import sys
    program = """
import sys
sys.modules["nesgpu_b200._host"] = None                  # an import of it fails
import torch
from nesgpu_b200 import base, microscaling
import modules.base, modules.binary
layer = base.PermutedLinear(8, 8, 2)
norm = base.PerturbedRMSNorm(8, 2)
microscaling.MicroscaledLinear(64, 64)
for call in (lambda: microscaling.quantize(torch.zeros(2, 64)), lambda: norm(torch.zeros(2, 8)), lambda: microscaling.linear(torch.zeros(2, 64), None)):
    try:
        call()
    except RuntimeError as e:
        print(e)
"""
    import os
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=600,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert run.returncode == 0, run.stderr
    said = run.stdout.splitlines()
    assert len(said) == 3 and all("python -m nesgpu_b200.build" in line for line in said[:2]) and "MicroscaledTensor" in said[2]


def test_build_makes_what_is_out_of_date(tmp_path, monkeypatch):
    """The extension module also when it was built for another PyTorch or Python, the library only for its sources; an extension
    module that cannot be built leaves the library in place."""
    import os
    from nesgpu_b200 import build as B
    done = []

    def write(path):
        with open(path, "w") as f:
            f.write("x")
        os.utime(path, (B._deps_mtime() + 10,) * 2)

    for name, value in (("LIB_DIR", "lib"), ("OBJ_DIR", "build"), ("LIB_PATH", "lib/l.so"), ("HOST_PATH", "_host.so"), ("HOST_TAG", "build/t")):
        monkeypatch.setattr(B, name, str(tmp_path / value))
    monkeypatch.setattr(B, "_compile", lambda src, verbose: (src, ""))
    monkeypatch.setattr(B, "_compile_host", lambda: "host.o")
    monkeypatch.setattr(B, "_link_library", lambda objs: (done.append("library"), write(B.LIB_PATH)))
    monkeypatch.setattr(B, "_link_host", lambda obj: (done.append(obj), write(B.HOST_PATH)))

    def made(**kw):
        del done[:]
        assert B.build(**kw) == B.LIB_PATH
        return list(done)

    assert made() == ["library", "host.o"] and made() == []
    monkeypatch.setattr(B, "_wanted_tag", lambda: "torch 9.9.9, python cpython-399")
    assert made() == ["host.o"] and made() == []
    os.remove(B.HOST_TAG)
    assert made() == ["host.o"] and made(force=True) == ["library", "host.o"]
    os.remove(B.HOST_PATH)
    assert made() == ["host.o"]

    def fails():
        raise RuntimeError("g++ failed")

    os.remove(B.LIB_PATH)
    monkeypatch.setattr(B, "_compile_host", fails)
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        B.build()
    assert os.path.exists(B.LIB_PATH) and B._built_tag() is None
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):             # and says so again
        B.build()


def test_outputs_over_one_another_are_refused():
    """Codes and scales, a norm's output and its residual, a product's output and its scratch; before anything reaches a device."""
    from nesgpu_b200 import _cabi as C
    f32, bf16, mx4, mx8 = 0, 1, 4, 8
    a, b, c, d, e, f = (n << 40 for n in range(1, 7))
    rows = 4 * 128 * 4                               # bytes of a (4, 128) fp32 matrix
    need = C.call("nes_mx_linear_fwd_scratch_bytes", 200, 64, 128, mx8)
    calls = [("nes_mx_quantize", (a, f32, b, b + 4 * 128 - 16, 4, 128, mx8, 0)),
             ("nes_mx_quantize", (a, f32, b, b, 4, 128, mx4, 0)),
             ("nes_rms_norm_fwd", (a, b, c, None, None, c, None, 4, 128, 0, 0, f32, 0, 1e-6, 0)),
             ("nes_rms_norm_fwd", (a, b, c, None, None, c + rows - 16, d, 4, 128, 0, 0, f32, mx8, 1e-6, 0)),
             ("nes_rms_norm_fwd", (a, b, c, None, None, d, c + rows - 1, 4, 128, 0, 0, f32, mx8, 1e-6, 0)),
             ("nes_rms_norm_fwd", (a, None, None, None, None, d, d + 16, 4, 128, 0, 0, f32, mx4, 1e-6, 0)),
             ("nes_mx_linear_fwd", (a, None, bf16, mx8, b, c, mx4, None, d + need - 32, f32, 200, 64, 128, d, need, 0))]
    for name, args in calls:
        with pytest.raises(C.NesError, match="overlap"):
            C.call(name, *args)
