"""The layers that use the microscaled operators, run one by one and together as a model uses them, against 64 bits.

Base products are exact up to the accumulation bound of the operators' own tests (well below 1e-6 of the output here);
the per-member terms come from the dense-noise kernels, whose stated bound is the relative 1e-4 used below.
"""
import numpy as np
import pytest
import torch

from gpu_util import REL_TOL, assert_close
from oracle import microscaled_ref as O
from test_gpu_microscaled import _check_linear

pytestmark = pytest.mark.gpu

MODES = {"mxfp4": ("mxfp4", "mxfp4"), "mxfp8": ("mxfp8", "mxfp8"), "mxfp8_mxfp4": ("mxfp8", "mxfp4")}


def _f64(t):
    return t.detach().cpu().double().numpy()


def _quantized(x64, form):
    codes, scales = O.quantize(x64, form)
    return O.values(codes, scales, form)


def _base(x64, layer, mode):
    """x W^T + b with both operands quantised as the layer's mode says."""
    a, w = MODES[mode]
    y, _ = O.linear(_quantized(x64, a), _quantized(_f64(layer.weight), w), None if layer.bias is None else _f64(layer.bias))
    return y


def _member_term(x64, layer, D, antithetic):
    noise, rows = _f64(layer.weight_noise), x64.shape[0]
    d, r = np.arange(rows) % D, np.arange(rows) // D
    sign = np.where(antithetic & (r >= (rows // D + 1) // 2), -1.0, 1.0)
    y = np.einsum("bi,boi->bo", x64, noise[d])
    if layer.bias is not None:
        y = y + _f64(layer.bias_noise)[d]
    return sign[:, None] * y


def _noisy(layer, scale=0.05, seed=3):
    layer.set_seed(seed)
    layer.set_noise(scale)
    return layer


def _rows(n, cols, seed, dtype=torch.float32):
    return (torch.randn(n, cols, generator=torch.Generator().manual_seed(seed)) * 2).to(dtype).cuda()


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("antithetic", [False, True])
@pytest.mark.parametrize("D,R,i,o", [(4, 1, 33, 7), (6, 4, 160, 48), (3, 50, 257, 130)])
def test_perturbed_linear(D, R, i, o, antithetic, bias, mode):
    from nesgpu_b200 import base
    layer = _noisy(base.PerturbedLinear(i, o, D, bias=bias, antithetic=antithetic, options={"tc": mode}).cuda())
    x = _rows(R * D, i, 1)
    assert_close(layer(x), torch.from_numpy(_base(_f64(x), layer, mode)), 1e-6, "plain")
    layer.perturbed_flag = True
    want = _base(_f64(x), layer, mode) + _member_term(_f64(x), layer, D, antithetic)
    assert_close(layer(x), torch.from_numpy(want), REL_TOL, "population")
    assert layer.last_path == mode


@pytest.mark.parametrize("mode", ["mxfp8", "mxfp8_mxfp4"])
def test_linear_layers_read_microscaled_inputs(mode):
    from nesgpu_b200 import base, microscaling as ms
    D = 5
    layer = _noisy(base.PerturbedLinear(96, 40, D, options={"tc": mode}).cuda())
    q = ms.quantize(_rows(15, 96, 2), "mxfp8")
    x64 = _f64(q.dequantize())
    assert_close(layer(q), torch.from_numpy(_base(x64, layer, mode)), 1e-6)      # quantising quantised values changes nothing
    layer.perturbed_flag = True
    assert_close(layer(q), torch.from_numpy(_base(x64, layer, mode) + _member_term(x64, layer, D, False)), REL_TOL)
    with pytest.raises(NotImplementedError, match="activations"):
        layer(ms.quantize(_rows(15, 96, 2), "mxfp4"))
    plain = base.PerturbedLinear(96, 40, D).cuda()
    with pytest.raises(NotImplementedError, match="microscaled"):
        plain(q)
    with pytest.raises(NotImplementedError, match="microscaled"):
        base.PermutedLinear(96, 40, D, options={"tc": "fp32"}).cuda()(q)


def test_sparse_perturbed_linear():
    from nesgpu_b200 import base
    D, i, o, k = 4, 72, 30, 3
    layer = base.SparsePerturbedLinear(i, o, D, options={"tc": "mxfp4"}, k=k).cuda()
    layer.allocate_memory()
    _noisy(layer)
    x = _rows(12, i, 4)
    layer.perturbed_flag = True
    dense = np.zeros((D, o, i))
    idx, val = layer.noise_indices.cpu().numpy(), _f64(layer.weight_noise)
    for d in range(D):
        for j in range(o):
            np.add.at(dense[d, j], idx[d, j], val[d, j])
    member = np.arange(12) % D
    want = _base(_f64(x), layer, "mxfp4") + np.einsum("bi,boi->bo", _f64(x), dense[member]) + _f64(layer.bias_noise)[member]
    assert_close(layer(x), torch.from_numpy(want), REL_TOL)
    assert layer(x[:0]).shape == (0, o)


@pytest.mark.parametrize("antithetic", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_layer(dtype, antithetic):
    from nesgpu_b200 import base
    D, n = 6, 200
    layer = _noisy(base.PerturbedRMSNorm(n, D, antithetic=antithetic).cuda(), 0.1)
    with torch.no_grad():
        layer.weight.add_(0.2 * torch.randn(n, generator=torch.Generator().manual_seed(0)).cuda())
    x, res = _rows(24, n, 5, dtype), _rows(24, n, 6, dtype)
    eps = float(np.float32(1e-6))
    half = torch.finfo(dtype).eps / 2
    want, _ = O.rms_norm(_f64(x), _f64(layer.weight), eps)
    assert np.all(np.abs(_f64(layer(x)) - want) <= (half + 2e-6) * np.abs(want))
    layer.perturbed_flag = True
    y, h = layer(x, res)
    want, h64 = O.rms_norm(_f64(x), _f64(layer.weight), eps, _f64(res), _f64(layer.weight_noise), antithetic)
    assert np.all(np.abs(_f64(y) - want) <= (half + 2e-6) * np.abs(want))
    assert torch.equal(h, (x.float() + res.float()).to(dtype)) and h.dtype == dtype
    with pytest.raises(RuntimeError, match="multiple of directions"):
        layer(x[:7])


def test_norm_layer_update_is_the_weighted_noise_sum():
    from nesgpu_b200 import base
    D, n = 64, 130
    layer = _noisy(base.PerturbedRMSNorm(n, D).cuda(), 0.1)
    w = torch.randn(D, generator=torch.Generator().manual_seed(1)).cuda()
    grad = layer.update(w)
    want = torch.from_numpy(_f64(w) @ _f64(layer.weight_noise))
    assert grad is layer.weight.grad
    assert_close(grad, want, 1e-5)
    layer.update(w, l2=0.5)
    assert_close(layer.weight.grad, 2 * want + 0.5 * layer.weight.detach().cpu().double(), 1e-5)
    # the same member draws the same gain noise wherever the population is split
    half = base.PerturbedRMSNorm(n, D // 2).cuda()
    half.set_member_offset(D // 2)
    _noisy(half, 0.1)
    full = _noisy(base.PerturbedRMSNorm(128, D).cuda(), 0.1)
    part = base.PerturbedRMSNorm(128, D // 2).cuda()
    part.set_member_offset(D // 2)
    _noisy(part, 0.1)
    assert torch.equal(part.weight_noise, full.weight_noise[D // 2:])


class Block(torch.nn.Module):
    """norm -> product -> ReLU -> product, and the residual, twice: 8-bit activations on the way into 4-bit weights."""

    def __init__(self, n, hidden, D, tc="mxfp8_mxfp4"):
        super().__init__()
        from nesgpu_b200 import base
        options = {"tc": tc}
        self.norms = torch.nn.ModuleList([base.PerturbedRMSNorm(n, D, options={"output": "mxfp8"}) for _ in range(2)])
        self.up = torch.nn.ModuleList([base.PerturbedLinear(n, hidden, D, options=options) for _ in range(2)])
        self.down = torch.nn.ModuleList([base.PerturbedLinear(hidden, n, D, options=options) for _ in range(2)])
        self.last = base.PerturbedRMSNorm(n, D)

    def forward(self, x):
        y, h = torch.zeros_like(x), x
        for norm, up, down in zip(self.norms, self.up, self.down):
            q, h = norm(y, h)
            y = down(torch.relu(up(q)))
        return self.last(y, h)[0]


def _block_oracle(m, x64, D, population):
    """The block in 64 bits, with every quantisation taken where the model takes it."""
    eps = float(np.float32(1e-6))
    y, h = np.zeros_like(x64), x64
    noise = (lambda l: _f64(l.weight_noise)) if population else (lambda l: None)
    for norm, up, down in zip(m.norms, m.up, m.down):
        q, h = O.rms_norm(y, _f64(norm.weight), eps, h, noise(norm))
        q = _quantized(q, "mxfp8")
        a = _base(q, up, "mxfp8_mxfp4") + (_member_term(q, up, D, False) if population else 0)
        a = np.maximum(a, 0)
        y = _base(a, down, "mxfp8_mxfp4") + (_member_term(a, down, D, False) if population else 0)
    return O.rms_norm(y, _f64(m.last.weight), eps, h, noise(m.last))[0]


def _block(D, n=96, hidden=160):
    from nesgpu_b200 import base
    torch.manual_seed(0)
    m = Block(n, hidden, D).cuda()
    pm = base.PerturbedModel(m, D)
    pm.set_seed(11)
    pm.set_noise(0.02)
    return m, pm


@pytest.mark.parametrize("population", [False, True])
def test_block_of_norms_and_products(population):
    """Together: a flipped rounding of one activation (a value within 1e-6 of a border) moves a code by a step, 2^-3 of that one
    value; with some 1e-5 of the values so near a border, the whole stays within 1e-2 of the 64-bit run in norm."""
    D = 4
    m, pm = _block(D)
    x = _rows(6 * D, 96, 8)
    with torch.no_grad():
        y = pm.forward(x) if population else m(x)
    want = _block_oracle(m, _f64(x), D, population)
    assert (np.linalg.norm(_f64(y) - want) / np.linalg.norm(want)) < 1e-2


def test_block_in_an_es_step():
    from nesgpu_b200 import es
    D = 16
    m, pm = _block(D)
    x, labels = _rows(10, 96, 9), torch.arange(10).cuda() % 96
    fitness, _ = es.es_step(pm, x, labels, D, noise_scale=0.02, chunk=10)
    assert fitness.shape == (D,) and torch.isfinite(fitness).all() and fitness.std() > 0
    for p in m.parameters():
        assert p.grad is not None and p.grad.shape == p.shape and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0


def test_microscaled_linear():
    from nesgpu_b200 import base, microscaling as ms
    torch.manual_seed(1)
    for bias in (True, False):
        src = base.PerturbedLinear(200, 70, 2, bias=bias).cuda()
        layer = ms.MicroscaledLinear.from_linear(src, "mxfp4", "mxfp8")
        x = _rows(9, 200, 3, torch.bfloat16)
        want = _base(_f64(x), src, "mxfp8_mxfp4")
        y = layer(x)
        assert y.dtype == torch.bfloat16 and y.shape == (9, 70)
        assert_close(layer(x, dtype=torch.float32), torch.from_numpy(want), 1e-6)
        assert_close(y, torch.from_numpy(want), 2.0 ** -8)
        other = ms.MicroscaledLinear(200, 70, bias).cuda()
        other.load_state_dict(layer.state_dict())
        assert torch.equal(other(x), y)
    assert not list(layer.parameters())


def test_two_graphs_replayed_at_once():
    """Norm and products captured into two graphs share no workspace: replayed on two streams over other inputs they give what
    the calls give one by one."""
    from nesgpu_b200 import microscaling as ms
    for rows in (1, 40, 300):
        w = ms.quantize(_rows(256, 512, 1))
        gain = torch.ones(512, device="cuda")
        xs = [_rows(rows, 512, 20 + i, torch.bfloat16) for i in range(2)]

        def call(x):
            q, h = ms.rms_norm(x, gain, residual=x, output="mxfp8")
            return ms.linear(q, w, dtype=torch.bfloat16), ms.linear(h, w, activations="mxfp4")

        call(xs[0])
        torch.cuda.synchronize()
        graphs, outs = [], []
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(x))
            graphs.append(g)
        for x in xs:
            x.copy_(torch.roll(x, 7, 1))
        want = [[t.clone() for t in call(x)] for x in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 40, 200, 900])
def test_calls_back_to_back(rows):
    """Weights quantised right before the product that reads them, activations quantised by the kernel before it, results consumed
    by the next call, in a row without a pause: what the same calls give one at a time."""
    from nesgpu_b200 import microscaling as ms
    W = [_rows(384, 512, 50 + i) for i in range(2)]
    V = [_rows(512, 384, 60 + i) for i in range(2)]
    X = [_rows(rows, 512, 70 + i, torch.bfloat16) for i in range(2)]

    def chain(i, pause):
        w = ms.quantize(W[i]); pause()
        y = ms.linear(X[i], w); pause()
        q = ms.rms_norm(y, output="mxfp8"); pause()
        v = ms.quantize(V[i], "mxfp8"); pause()
        z = ms.linear(q, v, dtype=torch.bfloat16); pause()
        return y, z, ms.linear(z, w, activations="mxfp4")

    want = [chain(i, torch.cuda.synchronize) for i in range(2)]
    torch.cuda.synchronize()
    got = [chain(i % 2, lambda: None) for i in range(40)]
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 2]):
            assert torch.equal(a, b), i


def test_calls_on_another_stream():
    from nesgpu_b200 import microscaling as ms
    w = ms.quantize(_rows(300, 640, 1), "mxfp8")
    x = _rows(500, 640, 2)
    want = ms.linear(ms.rms_norm(x, output="mxfp8"), w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            busy = busy @ busy * 1e-2                     # keeps the stream busy: work on any other one would overtake it
        x2 = x * 1.0 + 0 * busy[:500, :640].nan_to_num(0, 0, 0)
        got = ms.linear(ms.rms_norm(x2, output="mxfp8"), w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: the last rows are what they are by themselves."""
    from nesgpu_b200 import microscaling as ms
    rows, cols = 65544, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-8:] = _rows(8, cols, 1, torch.bfloat16)
    for form in ("mxfp4", "mxfp8"):
        q, part = ms.quantize(x, form), ms.quantize(x[-8:].contiguous(), form)
        assert torch.equal(q.codes[-8:], part.codes) and torch.equal(q.scales[-8:], part.scales)
        assert torch.equal(q.dequantize(torch.bfloat16)[-8:], part.dequantize(torch.bfloat16))
        assert torch.equal(q.elements()[-8:].view(torch.uint8), part.elements().view(torch.uint8))
    y, h = ms.rms_norm(x, residual=x, output="mxfp8")
    y8, h8 = ms.rms_norm(x[-8:].contiguous(), residual=x[-8:].contiguous(), output="mxfp8")
    assert torch.equal(y.codes[-8:], y8.codes) and torch.equal(h[-8:], h8)
    del y, h, q
    # activations, then weights, then the output of more than 2^31 bytes or elements
    w = ms.quantize(_rows(40, cols, 2))
    assert torch.equal(ms.linear(x, w)[-8:].float(), ms.linear(x[-8:].contiguous(), w, dtype=torch.float32).bfloat16().float())
    big = ms.quantize(x, "mxfp8")
    few = _rows(3, cols, 3)
    # the number of feature tiles decides how K is split, so eight rows by themselves are added in another order: the
    # bound of the products' own tests instead of equal bits
    _check_linear(ms.linear(few, big, activations="mxfp8")[:, -8:], _quantized(_f64(few), "mxfp8"), _quantized(_f64(x[-8:]), "mxfp8"),
                  None, torch.float32)
    del big
    a, b = ms.quantize(_rows(rows, 64, 4)), ms.quantize(_rows(cols, 64, 5))
    y = ms.linear(a, b, dtype=torch.bfloat16)
    want = ms.linear(a, ms.quantize(_rows(cols, 64, 5)[-8:].contiguous()), dtype=torch.bfloat16)
    assert torch.equal(y[:, -8:], want)


def test_graph_with_copies_fills_and_branches():
    """Captured calls that follow a copy, a fill, a join of two branches or another call: each waits for what it reads."""
    from nesgpu_b200 import microscaling as ms
    w = ms.quantize(_rows(512, 512, 1))
    given = _rows(600, 512, 2, torch.bfloat16)
    static, doubled = torch.empty_like(given), torch.empty_like(given)
    side = torch.cuda.Stream()

    def call():
        static.copy_(given)
        q, h = ms.rms_norm(static, residual=static, output="mxfp8")
        doubled.copy_(h)
        y = ms.linear(doubled, w, activations="mxfp4")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s = ms.linear(q, w, dtype=torch.bfloat16)
            back = q.dequantize(torch.bfloat16)
        z = ms.linear(y, w, dtype=torch.bfloat16)
        torch.cuda.current_stream().wait_stream(side)
        total = ms.rms_norm(z, residual=s)[1]
        z.zero_()
        return total, back, ms.rms_norm(back), ms.linear(z, w)

    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        given.copy_(torch.roll(given, 1 if i % 2 == 0 else -1, 0))
        for _ in range(3):
            graph.replay()
        ref = [torch.roll(t, 1, 0) if i % 2 == 0 else t for t in want]
        torch.cuda.synchronize()
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_calls_from_several_threads():
    import threading
    from nesgpu_b200 import microscaling as ms
    w = ms.quantize(_rows(256, 512, 1))
    xs = [_rows(rows, 512, 30 + rows, torch.bfloat16) for rows in (1, 40, 300)]

    def chain(x):
        q, h = ms.rms_norm(x, residual=x, output="mxfp8")
        return ms.linear(q, w, dtype=torch.bfloat16), ms.linear(h, w, activations="mxfp4")

    want = [[t.clone() for t in chain(x)] for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(x, ref, stream):
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = chain(x)
                if not all(torch.equal(a, b) for a, b in zip(got, ref)):
                    wrong.append(x.shape)

    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream()] * 2
    threads = [threading.Thread(target=work, args=(xs[i % 3], want[i % 3], s)) for i, s in enumerate(streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
