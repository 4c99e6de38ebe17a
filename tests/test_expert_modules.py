"""Int4Linear and Int4Experts: against their formulas in 64 bits, as they are served; the operators around experts as they are trained."""
import copy

import pytest
import torch

import fp6_llm_amd as fp6
from fp6_llm_amd import int4
from fp6_llm_amd.module import FPxGatedLinear, FPxLinear, Int4Experts, Int4Linear
from test_experts import Plan64, route
from test_int4 import HALF, TINY, Weight, d, gated64, plain, product64, randn, within

DEV = "cuda:0"
gpu = pytest.mark.gpu


def triple(w):
    return w.codes, w.scales, w.zeros


def pairs64(gate, up):
    """Rows of gate and up, [F, ...] each, in pair order."""
    return fp6.gate_up_pairs(gate, up)


def layer64(gate, up, down, x, index, weights, act, dtype):
    """The layer and how far it may be off: the hidden rows are rounded to the activations' type, their products are float32 sums, which are added up in float32 and rounded once."""
    T, k = index.shape
    extra = 30 if dtype == torch.bfloat16 else 1   # (products of few bf16 rows: 143 at most stands for each of q and z, 5 on average)
    out, tol = torch.zeros(T, x.shape[1], dtype=torch.float64), torch.zeros(T, x.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for t in range(T):
        for j in range(k):
            e = int(index[t, j])
            if not 0 <= e < gate.E:
                continue
            y, err = product64(pairs64(gate.w[e], up.w[e]), x[t:t + 1])
            h, et = gated64(y, extra * err, act, dtype)
            z, ez = h @ down.w[e].t(), et @ down.w[e].abs().t() + extra * (down.IC + 3) * 2.0 ** -23 * (h.abs() @ down.w[e].abs().t())
            ez = ez + 2.0 ** -24 * z.abs()
            w = float(weights[t, j])
            out[t] += w * z[0]
            tol[t] += abs(w) * ez[0]
            mag[t] += abs(w) * z[0].abs()
    return out, (tol + k * 2.0 ** -23 * mag) * (1 + HALF[dtype]) + HALF[dtype] * out.abs() + TINY[dtype]


@gpu
@pytest.mark.parametrize("T,k,E,F,K,group,zeros,type,act,drop", [(1, 2, 8, 96, 128, 128, False, "fp16", "silu", 0.0), (5, 3, 4, 160, 96, 32, True, "bf16", "gelu", 0.3), (40, 2, 3, 64, 288, 64, True, "fp16", "gelu_tanh", 0.1),
                                                                 (130, 1, 2, 352, 160, 128, True, "bf16", "silu", 0.0), (64, 4, 16, 32, 64, 96, False, "fp16", "silu", 0.0)])
def test_experts_layer(T, k, E, F, K, group, zeros, type, act, drop):
    gate, up, down = Weight(1, F, K, group, zeros, type, E), Weight(2, F, K, group, zeros, type, E), Weight(3, K, F, group, zeros, type, E)
    layer = Int4Experts.from_codes(triple(gate), triple(up), triple(down), group, act)
    index, x = route(T, T, k, E, drop), randn(4, T, K, dtype=gate.dtype)
    weights = torch.rand(T, k, generator=torch.Generator().manual_seed(5)).to(DEV)
    want, tol = layer64(gate, up, down, x, index, weights, act, gate.dtype)
    got = layer(x, index, weights)
    assert got.dtype == gate.dtype
    within(got, want, tol)
    # more dimensions, other types of the input, no weights
    assert torch.equal(layer(x.view(T, 1, K), index.view(T, 1, k), weights.view(T, 1, k)), got.view(T, 1, K))
    assert torch.equal(layer(x.float(), index.int(), weights.double()), got)
    within(layer(x, index), *layer64(gate, up, down, x, index, torch.ones(T, k), act, gate.dtype))
    assert layer(x[:0], index[:0], weights[:0]).shape == (0, K)


@gpu
def test_experts_layer_in_a_graph():
    """One token at a time, as it is decoded: index, weights and input change between the replays."""
    E, F, K, k = 8, 256, 192, 2
    layer = Int4Experts.from_float(*(randn(i, E, *s, dtype=torch.float32, scale=0.1) for i, s in enumerate(((F, K), (F, K), (K, F)))), group=64, zeros=True)
    for T in (1, 3, 200):
        x, index, weights = randn(1, T, K), route(1, T, k, E), torch.rand(T, k, device=DEV)
        layer(x, index, weights)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer(x, index, weights)
        for seed in range(2, 6):
            x.copy_(randn(seed, T, K)), index.copy_(route(seed, T, k, E, 0.2)), weights.copy_(torch.rand(T, k))
            want = layer(x, index, weights)
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_linear_layer(type):
    w = Weight(7, 272, 288, 96, True, type)
    b = randn(1, 272, dtype=w.dtype)
    layer = Int4Linear.from_codes(*triple(w), 96, b)
    for shape in ((5, 288), (2, 3, 288), (288,), (0, 288), (70, 288)):
        x = randn(2, *shape, dtype=w.dtype)
        got = layer(x)
        assert got.shape == shape[:-1] + (272,) and got.dtype == w.dtype
        y, err = product64(w.w, x.reshape(-1, 288), b, extra=w if type == "bf16" else None)
        within(got.reshape(-1, 272), *plain(y, err, w.dtype))
    buffer = randn(3, 8 * 288 + 1, dtype=w.dtype)
    assert torch.equal(layer(buffer[1:].view(8, 288)), layer(buffer[1:].clone().view(8, 288)))
    assert torch.equal(layer(x.float()), layer(x))


@gpu
@pytest.mark.parametrize("zeros", [False, True])
def test_quantized_layers_are_near_the_float_ones(zeros):
    weight = randn(1, 256, 512, dtype=torch.float32, scale=0.05)
    layer = Int4Linear.from_float(weight, 64, zeros)
    x = randn(2, 9, 512)
    y = d(x) @ d(weight).t()
    # a weight is off by a step of its group at most (half a step, half of the zero point's), and a step is a fifteenth of a range that normal numbers of 64 do not leave 9 sigma wide
    assert ((d(layer(x)) - y).abs() <= d(x).abs().sum(1, keepdim=True) * 0.05 * 9 / 15 + 0.01).all()


def test_modules_on_the_host():
    w = randn(1, 64, 96, dtype=torch.float32, device="cpu")
    layer = Int4Linear.from_float(w, 32, True, torch.zeros(64, dtype=torch.float16))
    other = Int4Linear(96, 64, 32, True, torch.ones(64, dtype=torch.float16))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.weight_native, layer.weight_native) and torch.equal(other.weight_scales, layer.weight_scales) and torch.equal(other.bias, layer.bias)
    assert all(torch.equal(a, b) for a, b in zip(copy.deepcopy(layer).state_dict().values(), layer.state_dict().values()))
    for cast in (torch.nn.Sequential(layer).float(), torch.nn.Sequential(layer).bfloat16(), torch.nn.Sequential(layer).double()):
        assert cast[0].weight_scales.dtype == torch.float16 and cast[0].bias.dtype == torch.float16 and cast[0].weight_native.dtype == torch.int32
    E, F, K = 3, 64, 96
    ws = [randn(i, E, *s, dtype=torch.bfloat16, device="cpu") for i, s in enumerate(((F, K), (F, K), (K, F)))]
    experts = Int4Experts.from_float(*ws, group=32)
    assert experts.dtype == torch.bfloat16 and "experts=3" in repr(experts) and "out_features=64" in repr(layer)
    again = Int4Experts(K, F, E, 32, dtype=torch.bfloat16)
    again.load_state_dict(experts.state_dict())
    assert torch.equal(again.gate_up_native, experts.gate_up_native) and torch.nn.Sequential(again).half()[0].down_scales.dtype == torch.bfloat16
    # an expert's part is that of its own two matrices in pair order
    g, u = (int4.int4_quantize(w[1], 32) for w in ws[:2])
    one = int4.int4_pack_native(*(None if a is None else fp6.gate_up_pairs(a, b) for a, b in zip(g, u)), 32)
    assert torch.equal(experts.gate_up_native[1], one[0]) and torch.equal(experts.gate_up_scales[1], one[1])


def test_refusals_of_the_modules():
    for args in ((96, 40), (90, 64), (96, 64, 48), (96, 64, 0)):
        with pytest.raises(ValueError):
            Int4Linear(*args)
    with pytest.raises(ValueError):
        Int4Linear(96, 64, dtype=torch.float32)
    with pytest.raises(ValueError):
        Int4Linear(96, 64, bias=torch.zeros(64))
    for args in ((96, 48, 2), (80, 64, 2), (96, 64, 0), (96, 64, 2000), (96, 64, 2, 40)):
        with pytest.raises(ValueError):
            Int4Experts(*args)
    with pytest.raises(ValueError):
        Int4Experts(96, 64, 2, activation="relu")
    layer, experts = Int4Linear(96, 64), Int4Experts(96, 64, 2)
    x = torch.zeros(4, 96, dtype=torch.float16)
    index, weights = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    for bad in (lambda: layer(x[:, :64]), lambda: layer(x.clone().requires_grad_()), lambda: experts(x[:, :64], index), lambda: experts(x, index[0]), lambda: experts(x, index[:3]), lambda: experts(x, index, weights[:, :1]),
                lambda: experts(x.clone().requires_grad_(), index), lambda: experts(x, index, weights.clone().requires_grad_()), lambda: layer(x), lambda: experts(x, index)):   # (the last two: not on a GPU)
        with pytest.raises(ValueError):
            bad()
    q = [int4.int4_quantize(torch.zeros(2, *s, dtype=torch.float16), 32) for s in ((64, 96), (64, 96), (96, 64))]
    with pytest.raises(ValueError):
        Int4Experts.from_codes(q[0], q[1], q[1], 32)
    with pytest.raises(ValueError):
        Int4Experts.from_codes(q[0], int4.int4_quantize(torch.zeros(2, 64, 96), 32, True), q[2], 32)


@gpu
def test_experts_as_they_are_trained():
    """Rows sorted, each expert's share through its own differentiable block, summed back with the router's weights: gradients of input and weights against a mixture of dense products in 64 bits."""
    T, k, E, H = 23, 2, 3, 256
    index = route(3, T, k, E, 0.1)
    x, w = randn(1, T, H, dtype=torch.float32).requires_grad_(), torch.rand(T, k, device=DEV).requires_grad_()
    mats = [randn(10 + e, H, H, dtype=torch.float32, scale=0.05) for e in range(E)]
    rows, plan = fp6.expert_sort(x, index, E)
    offsets = plan.offsets.tolist()
    parts = [torch.tanh(rows[a:b] @ m.t()) for a, b, m in zip(offsets, offsets[1:], mats)] + [rows[offsets[-1]:]]
    out = fp6.expert_combine(torch.cat(parts), plan, w)
    g = randn(2, T, H, dtype=torch.float32)
    gx, gw = torch.autograd.grad(out, (x, w), g)
    x64, w64 = d(x).requires_grad_(), d(w).requires_grad_()
    want = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if 0 <= (e := int(index[t, j])) < E:
                want[t] = want[t] + w64[t, j] * torch.tanh(x64[t] @ d(mats[e]).t())
    wx, ww = torch.autograd.grad(want, (x64, w64), d(g))
    # float32 products of 256 terms on both ways, a hyperbolic tangent to 2^-20: 2^-13 of typical magnitudes (products of 256 normal numbers and 0.05: below 8; gradients below 2^5)
    for got, exact, size in ((out, want.detach(), 2.0), (gx, wx, 32.0), (gw, ww, 512.0)):
        within(got, exact, torch.full_like(exact, size * 2.0 ** -13))


@gpu
def test_experts_of_the_other_formats():
    """Frozen FPx blocks, one for each expert, between the sort and the sum: the gradient reaches the tokens through them."""
    T, k, E, K, F = 30, 2, 2, 256, 256
    index = route(4, T, k, E)
    gated = [FPxGatedLinear.from_float(randn(e, F, K, scale=0.06), randn(e + 9, F, K, scale=0.06)) for e in range(E)]
    down = [FPxLinear.from_float(randn(e + 20, K, F, scale=0.06)) for e in range(E)]
    for layer in down:
        layer.input_gradient = True
    x = randn(1, T, K).requires_grad_()
    w = torch.rand(T, k, device=DEV).requires_grad_()

    def mixture(x, w):
        rows, plan = fp6.expert_sort(x, index, E)
        o = plan.offsets.tolist()
        return fp6.expert_combine(torch.cat([down[e](gated[e](rows[o[e]:o[e + 1]])) for e in range(E)]), plan, w)
    g = randn(2, T, K)
    gx, gw = torch.autograd.grad(mixture(x, w), (x, w), g)

    def alone(t):   # a token by itself, its experts one after another
        xt = x[t:t + 1].detach().requires_grad_()
        ys = [down[int(e)](gated[int(e)](xt)) for e in index[t]]
        return torch.autograd.grad(ys, xt, [g[t:t + 1] * float(w[t, j]) for j in range(k)])[0], torch.stack([(d(y) * d(g[t:t + 1])).sum() for y in ys])
    for t in range(0, T, 7):
        ax, aw = alone(t)
        # (the same kernels on other batches: float16 roundings of the output's gradient, the product's, the sum's)
        assert ((d(gx[t]) - d(ax[0])).abs() <= 8 * HALF[torch.float16] * d(ax[0]).abs().max() + 1e-5).all()
        assert ((d(gw[t]) - aw).abs() <= 8 * HALF[torch.float16] * aw.abs().max() + 1e-2).all()
