"""The modules over the operators around the linear layer: FPxGatedLinear, LowRankAdapters, and FPxLinear with an input gradient.  Tolerances are counted as in test_operators.py."""
import pytest
import torch

import fp6_llm_amd as fp6
from fp6_llm_amd.module import _CROSSOVER_LIBRARY as LONG, FPxGatedLinear, FPxLinear, LowRankAdapters
from test_operators import DEV, HALF, TINY, Weight, adapters64, d, gated64, gpu, halves, pairs, preacts, randn, slope64, act64, sum_error, within


def layer(w, bias=None):
    m = FPxLinear(w.IC, w.OC, w.E, w.M, bias, group_scales=w.exps is not None).to(DEV)
    m.weight_native.copy_(w.native)
    m.scales.copy_(w.scales)
    if w.exps is not None:
        m.group_exps.copy_(w.exps)
    return m


def block(w, act="silu", bias=None):
    m = FPxGatedLinear(w.IC, w.OC // 2, w.E, w.M, act, bias, group_scales=w.exps is not None).to(DEV)
    m.weight_native.copy_(w.native)
    m.scales.copy_(w.scales)
    if w.exps is not None:
        m.group_exps.copy_(w.exps)
    return m


@pytest.mark.parametrize("groups", [False, True])
def test_gated_block_from_two_layers_holds_their_rows_in_pairs(groups):
    g = torch.Generator().manual_seed(1)
    gate, up = (torch.randn(256, 192, generator=g) for _ in range(2))
    biases = [torch.randn(256, generator=g).half() for _ in range(2)]
    both = FPxLinear.from_float(fp6.gate_up_pairs(gate, up), 2, 2, group_scales=groups)
    a = FPxGatedLinear.from_layers(*(FPxLinear.from_float(t, 2, 2, b, group_scales=groups) for t, b in zip((gate, up), biases)), activation="gelu")
    b = FPxGatedLinear.from_float(gate, up, 2, 2, "gelu", biases, group_scales=groups)
    for m in (a, b):
        assert (m.in_features, m.out_features, m.activation) == (192, 256, "gelu")
        assert torch.equal(m.weight_native, both.weight_native) and torch.equal(m.scales, both.scales) and torch.equal(m.bias, fp6.gate_up_pairs(*biases))
        assert (m.group_exps is None) == (not groups) and (not groups or torch.equal(m.group_exps, both.group_exps))
    b.load_state_dict(a.state_dict())
    assert set(a.state_dict()) == {"weight_native", "scales", "bias"} | ({"group_exps"} if groups else set()) and not list(a.parameters())


def test_refusals_of_the_modules():
    lin = lambda i=64, o=256, **kw: FPxLinear(i, o, **kw)   # noqa: E731
    for pair in ((lin(), lin(o=512)), (lin(), lin(i=128)), (lin(), lin(exponent=2)), (lin(), lin(bias=torch.zeros(256).half())), (lin(group_scales=True), lin())):
        with pytest.raises(ValueError):
            FPxGatedLinear.from_layers(*pair)
    for args in ((64, 64), (32, 128), (64, 0), (64, 128, 3, 2, "relu")):
        with pytest.raises(ValueError):
            FPxGatedLinear(*args)
    for args in ((64, 128, 1, 8), (32, 256, 1, 8), (64, 256, 0, 8), (64, 256, 1, 0), (64, 256, 1, 257)):
        with pytest.raises(ValueError):
            LowRankAdapters(*args)
    ad = LowRankAdapters(64, 256, 3, 12)
    assert ad.rank == 16
    a, b = torch.randn(12, 64), torch.randn(256, 12)
    for args in ((3, a, b), (-1, a, b), (0, a[:, :32], b), (0, a, b[:128]), (0, a[:8], b), (0, torch.randn(17, 64), torch.randn(256, 17)), (0, [a], [b, b]), (0, [], []), (0, [a, a], [b[:100], b[100:, :8]])):
        with pytest.raises(ValueError):
            ad.set(*args)
    with pytest.raises(ValueError):
        ad.clear(3)
    assert not ad.lora_a.any() and not ad.scaling.any()
    m, x, idx = lin(), torch.zeros(2, 64).half(), torch.zeros(2, dtype=torch.int32)
    for args in ((x, ad), (x, None, idx), (x, lin(), idx), (x, LowRankAdapters(128, 256, 1, 8), idx), (x, ad, idx[:1]), (x, ad, idx.reshape(1, 2)), (x.reshape(1, 2, 64), ad, idx.reshape(2, 1)),
                 (x[:, :32], ad, idx), (x.clone().requires_grad_(), ad, idx)):
        with pytest.raises(ValueError):
            m(*args)
    with pytest.raises(ValueError):
        FPxGatedLinear(64, 128)(torch.zeros(2, 128).half())   # (128 features would also be twice as many rows)
    biased = FPxGatedLinear(64, 128, bias=torch.zeros(256).half().requires_grad_())
    with pytest.raises(ValueError):
        biased(x)


def test_adapters_of_a_fused_layer_reach_their_parts():
    g = torch.Generator().manual_seed(2)
    ad = LowRankAdapters(64, 768, 2, 16)
    parts = [(torch.randn(r, 64, generator=g).half(), torch.randn(256, r, generator=g).half()) for r in (4, 2, 8)]
    ad.set(1, torch.ones(16, 64), torch.ones(768, 16), 3.0)
    ad.set(1, [a for a, _ in parts], [b for _, b in parts], 0.5)
    want = torch.cat([b.double() @ a.double() for a, b in parts])
    assert torch.equal(ad.lora_b[1].double() @ ad.lora_a[1].double(), want) and ad.scaling.tolist() == [0.0, 0.5]
    ad.clear(1)
    assert not ad.lora_a.any() and not ad.lora_b.any() and not ad.scaling.any()


def test_adapters_keep_their_types_in_a_model_that_is_cast():
    ad = LowRankAdapters(64, 256, 2, 8)
    ad.set(0, torch.randn(8, 64), torch.randn(256, 8), 1 / 3)
    want = {k: t.clone() for k, t in ad.state_dict().items()}
    for cast in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu", torch.float32)):
        assert cast(torch.nn.Sequential(ad))[0] is ad
        assert all(t.dtype == want[k].dtype and torch.equal(t, want[k]) for k, t in ad.state_dict().items())


@gpu
def test_indexes_that_are_views():
    w = Weight(1, 3, 2, 256, 128)
    m, ad = layer(w), LowRankAdapters(128, 256, 3, 8).to(DEV)
    for i in range(3):
        ad.set(i, randn(i, 8, 128, scale=0.1), randn(i + 5, 256, 8))
    x, table = randn(7, 6, 4, 128), torch.randint(-1, 3, (6, 2), generator=torch.Generator().manual_seed(1)).int().to(DEV)
    want = m(x, ad, table[:, 1].reshape(6, 1).repeat(1, 4).contiguous())
    assert torch.equal(m(x, ad, table[:, 1:].expand(6, 4)), want)
    assert torch.equal(m(x[:, 0], ad, table[:, 1]), m(x[:, 0].contiguous(), ad, table[:, 1].contiguous()))


@gpu
@pytest.mark.parametrize("N,act", [(1, "silu"), (23, "gelu"), (300, "gelu_tanh")])
def test_gated_module_is_its_function_and_differentiable(N, act):
    w, b = Weight(N, 2, 2, 512, 320, True), randn(1, 512, scale=0.3)
    m = block(w, act, b)
    x, dh = randn(2, N, 320), randn(3, N, 256, scale=0.1)
    pre = torch.empty(N, 512, device=DEV)
    h = fp6.gated_forward_native(2, 2, x, w.native, w.scales, 512, act, preact=pre, group_exps=w.exps, bias=b)
    dx = fp6.gated_backward_native(2, 2, dh, pre, w.native, w.scales, 320, act, group_exps=w.exps)[0]
    assert torch.equal(m(x), h) and not m(x).requires_grad
    leaf = x.clone().requires_grad_()
    y = m(leaf)
    assert torch.equal(y, h)
    y.backward(dh)
    assert torch.equal(leaf.grad, dx)
    with torch.no_grad():
        assert not m(leaf).requires_grad
    # more dimensions, a float32 leaf (whose cast autograd differentiates), a gradient of stride zero
    wide = x.float().reshape(1, N, 320).requires_grad_()
    y = m(wide)
    assert y.shape == (1, N, 256) and torch.equal(y.reshape(N, 256), h)
    y.sum().backward()
    ones = fp6.gated_backward_native(2, 2, torch.ones_like(dh), pre, w.native, w.scales, 320, act, group_exps=w.exps)[0]
    assert wide.grad.dtype == torch.float32 and torch.equal(wide.grad.reshape(N, 320), ones.float())
    # once only
    y = m(leaf)
    (g,) = torch.autograd.grad(y, leaf, dh.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


@gpu
@pytest.mark.parametrize("N,dequant_above", [(1, "auto"), (40, "auto"), (200, None), (200, 100)])
def test_input_gradient_of_the_linear_layer(N, dequant_above):
    w, b = Weight(N, 3, 2, 768, 448), randn(1, 768)
    m = layer(w, b)
    m.dequant_above = dequant_above
    x, dy = randn(2, N, 448), randn(3, N, 768)
    want = m(x)
    leaf = x.clone().requires_grad_()
    if dequant_above != 100:   # (above it the library's product is differentiated, as it always was)
        assert not m(leaf).requires_grad
    m.input_gradient = True
    y = m(leaf)
    assert y.requires_grad and torch.equal(y, want) and not m(x).requires_grad
    y.backward(dy)
    assert torch.equal(leaf.grad, fp6.linear_input_grad_native(3, 2, dy, w.native, w.scales, 448))
    # against a difference: the layer is linear, so <dy, m(x + v) - m(x)> is <dx, v> but for the roundings of the two outputs, of x + v and of dx
    v = randn(4, N, 448)
    xv = (x + v)
    lhs = (d(dy) * (d(m(xv)) - d(want))).sum()
    moved = d(xv) - d(x)
    (y0, e0), (y1, e1) = preacts(w, x, b), preacts(w, xv, b)
    base = 2 * HALF if dequant_above == 100 else 0   # (fp16 weights: value times scale is rounded once more; and a bias added to a rounded product)
    mags = (d(x).abs() + d(xv).abs()) @ w.w.abs().t() + 2 * d(b).abs()
    tol = (d(dy).abs() * (e0 + e1 + HALF * (y0.abs() + y1.abs()) * (1 + HALF) + 2 * TINY + base * mags)).sum()
    mag = d(dy).abs() @ w.w.abs()
    tol = tol + (moved.abs() * ((sum_error(768) + HALF) * mag + HALF * d(leaf.grad).abs() + 2 * TINY)).sum()
    assert abs(lhs - (d(leaf.grad) * moved).sum()) <= tol
    m.bias.requires_grad_()
    with pytest.raises(ValueError):
        m(leaf)


@gpu
@pytest.mark.parametrize("N", [3, 20, 300])
def test_one_feed_forward_layer_as_it_is_trained_and_as_it_is_served(N):
    """Queries, keys and values with a request's adapters, the gated block and the projection down with adapters; and the gradient through block and projection.  Every stage is held to
    its formula in 64 bits on the values that went into it."""
    H, F, slots = 512, 768, 4
    qkv, gu, down = Weight(1, 3, 2, 3 * H, H), Weight(2, 2, 2, 2 * F, H, True), Weight(3, 3, 2, H, F)
    mq, mg, md = layer(qkv), block(gu), layer(down)
    ads, oad = LowRankAdapters(H, 3 * H, slots, 40).to(DEV), LowRankAdapters(F, H, slots, 8).to(DEV)
    for i in range(3):
        ads.set(i, [randn(10 * i + j, 8 * (i + 1) if j == 0 else 8, H, scale=H ** -0.5) for j in range(3)],
                [randn(10 * i + j + 5, H, 8 * (i + 1) if j == 0 else 8, scale=0.2) for j in range(3)], 0.5 + i)
        oad.set(i, randn(40 + i, 8, F, scale=F ** -0.5), randn(50 + i, H, 8, scale=0.2), 1.0)
    index = (torch.arange(N, device=DEV) % 5 - 1).int()   # (-1: none; 3: a slot that nobody has set)
    x = randn(4, N, H)
    y = mq(x.reshape(1, N, H), ads, index.reshape(1, N)).reshape(N, 3 * H)
    want, tol = adapters64(qkv, x, None, ads.lora_a, ads.lora_b, ads.scaling, index.cpu())
    within(y, want, tol, "qkv")
    hidden = y[:, 2 * H:]   # (strided: one part of a fused layer's output)
    h = mg(hidden)
    within(h, *gated64(gu, hidden, None, "silu")[2:], "block")
    out = md(h, oad, index)
    want, tol = adapters64(down, h, None, oad.lora_a, oad.lora_b, oad.scaling, index.cpu())
    within(out, want, tol, "down")
    assert torch.equal(out[index < 0], md(h)[index < 0])   # (the bits of the layer alone)

    md.input_gradient = True
    leaf, dy = hidden.detach().clone().requires_grad_(), randn(7, N, H, scale=0.1)
    hh = mg(leaf)
    hh.retain_grad()
    md(hh).backward(dy)
    mag = d(dy).abs() @ down.w.abs()
    dh = d(dy) @ down.w
    within(hh.grad, dh, (sum_error(H + 3) + HALF) * mag + TINY * down.w.abs().sum(0) + HALF * dh.abs() + TINY, "dh")
    p, err = preacts(gu, hidden, None)
    (g, u), (eg, eu), dd = halves(p), halves(err), d(hh.grad)
    dp = pairs(dd * u * slope64("silu", g), dd * act64("silu", g))
    ep = pairs(dd.abs() * (1.3 * eg * u.abs() + 1.13 * eu + 2.0 ** -17 * u.abs()), dd.abs() * (1.13 * eg + 2.0 ** -17 * g.abs())) + (HALF + sum_error(2 * F)) * dp.abs() + TINY
    dx = dp @ gu.w
    within(leaf.grad, dx, (ep @ gu.w.abs()) * (1 + HALF) + HALF * dx.abs() + TINY, "dx")


@gpu
def test_slots_written_between_the_replays_of_a_graph():
    w = Weight(1, 3, 2, 512, 256)
    m, ad = layer(w), LowRankAdapters(256, 512, 2, 16).to(DEV)
    x, index = randn(1, 20, 256), (torch.arange(20, device=DEV) % 3 - 1).int()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        m(x, ad, index)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = m(x, ad, index)
        for i in range(3):
            ad.set(i % 2, randn(i, 9, 256, scale=0.1), randn(i + 9, 512, 9), 0.5)
            if i == 2:
                ad.clear(1)
            index.copy_(index.roll(1))
            graph.replay()
            assert torch.equal(y, m(x, ad, index))
            want, tol = adapters64(w, x, None, ad.lora_a, ad.lora_b, ad.scaling, index.cpu())
            within(y, want, tol)


@gpu
def test_captured_training_step():
    """Forward and backward of block and projection in one graph replay to the eager gradients."""
    gu, down = Weight(2, 2, 2, 512, 320, True), Weight(3, 3, 2, 512, 256)
    mg, md = block(gu), layer(down)
    md.input_gradient = True
    x, dy = randn(1, 40, 320), randn(2, 40, 512)

    def step(t):
        return torch.autograd.grad(md(mg(t)), t, dy)[0]
    if fp6._ext is None:   # (nothing says there where a gradient would go)
        pytest.skip("a differentiable call is captured with the extension alone")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(x.detach().clone().requires_grad_())
        leaf = x.detach().clone().requires_grad_()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            g = step(leaf)
        for seed in range(3):
            with torch.no_grad():
                leaf.copy_(randn(10 + seed, 40, 320))
            want = step(leaf.detach().clone().requires_grad_())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(g, want)


@gpu
def test_a_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    mg, md = block(Weight(2, 2, 2, 512, 320)), layer(Weight(3, 3, 2, 512, 320))
    md.input_gradient = True
    leaf = randn(1, 8, 320).requires_grad_()
    eager = [mg(leaf), md(leaf)]
    stream, buf = torch.cuda.Stream(), torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        buf.add_(1)
        for m in (mg, md):
            for t in (leaf, leaf * 1, leaf.float()):
                with pytest.raises(RuntimeError):
                    m(t)
        with torch.no_grad():   # (no gradient, nothing to refuse)
            y = mg(leaf)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, eager[0]) and (buf == 1).all()
    eager[0].sum().backward()
    assert leaf.grad is not None


@gpu
@pytest.mark.parametrize("N", [1, 5, 40])
def test_gradients_that_start_between_two_16_byte_boundaries(N):
    """The gradient of a concatenation's later part is a view into the whole one's, at whatever place the part has."""
    mg, md = block(Weight(2, 2, 2, 512, 320, True)), layer(Weight(3, 3, 2, 512, 320))
    md.input_gradient = True
    for m in (mg, md):
        x, dy = randn(1, N, 320), randn(2, N, m.out_features, scale=0.1)
        leaf = x.clone().requires_grad_()
        m(leaf).backward(dy)
        other, first = x.clone().requires_grad_(), torch.ones(1, dtype=torch.float16, device=DEV, requires_grad=True)
        torch.cat([first, m(other).flatten()]).backward(torch.cat([first.detach(), dy.flatten()]))
        assert torch.equal(other.grad, leaf.grad) and first.grad == 1


def splits_asked_for(monkeypatch, name):
    """The splitK that a module hands to a function of ops, call by call (its result is zeros of the right shape)."""
    asked = []

    def stand_in(E, M, x, native, scales, OC, *args, **kw):
        asked.append(kw.get("splitK", args[0] if name == "linear_forward_native" else args[1] if name == "gated_forward_native" else args[4]))
        return torch.zeros(x.shape[0], OC // 2 if name == "gated_forward_native" else OC, dtype=torch.float16)
    from fp6_llm_amd import module
    monkeypatch.setattr(module if name == "linear_forward_native" else module.ops, name, stand_in)
    return asked


def test_split_of_a_gated_block_is_for_batches_below_a_long_prompt(monkeypatch):
    asked = splits_asked_for(monkeypatch, "gated_forward_native")
    m = FPxGatedLinear(64, 128, split_k=4)
    for n in (1, LONG - 1, LONG, 9000):
        m(torch.zeros(n, 64).half())
    m(torch.zeros(1536, 2, 64).half())
    for none in (None, 0):
        FPxGatedLinear(64, 128, split_k=none)(torch.zeros(1, 64).half())
    assert asked == [4, 4, None, None, None, None, None]


def test_split_of_a_layer_holds_with_adapters(monkeypatch):
    asked = splits_asked_for(monkeypatch, "adapter_forward_native")
    plain = splits_asked_for(monkeypatch, "linear_forward_native")
    ad = LowRankAdapters(64, 256, 1, 8)
    for kw in (dict(split_k=2), dict(split_k=2, dequant_above=None), dict()):
        m = FPxLinear(64, 256, **kw)
        for n in (1, LONG - 1, LONG):
            x, index = torch.zeros(n, 64).half(), torch.zeros(n, dtype=torch.int32)
            m(x, ad, index), m(x)
    assert [s for s in asked[:6]] == [2, 2, None, 2, 2, 2] and asked[6:] == [None] * 3
    assert [p == (a or p) for a, p in zip(asked, plain)] == [True] * 9   # (None: the heuristic's, which the layer asks itself)


@gpu
@pytest.mark.parametrize("N", [3, 40])
def test_a_layer_with_adapters_is_the_layer_where_there_are_none(N):
    """Its split, and a bias that torch has to add (a float32 one, a strided one), are the same with adapters as without."""
    w = Weight(1, 3, 2, 512, 1344)
    ad, x, index = LowRankAdapters(1344, 512, 2, 8).to(DEV), randn(1, N, 1344), (torch.arange(N, device=DEV) % 3 - 1).int()
    for i in range(2):
        ad.set(i, randn(i, 8, 1344, scale=0.1), randn(i + 5, 512, 8))
    biases = [None, randn(2, 512), randn(2, 512).float(), randn(2, 512, 2)[:, 0]]
    for bias in biases:
        for split in (None, 2, 3):
            m = layer(w, bias)
            m.split_k = split
            y, alone = m(x, ad, index), m(x)
            assert y.dtype == alone.dtype and torch.equal(y[index < 0], alone[index < 0]), (bias is None or bias.dtype, split)
            want, tol = adapters64(w, x, bias, ad.lora_a, ad.lora_b, ad.scaling, index.cpu())
            extra = 0 if bias is None else 2 * d(bias).abs()   # (a bias behind the product: what is rounded before it is of the outputs without it, and one rounding more)
            within(y, want, tol + HALF * (want.abs() + extra) * (1 + 2 * HALF) + TINY)


def test_biases_that_a_block_cannot_take():
    for bias in (torch.zeros(256), torch.zeros(256).bfloat16(), torch.zeros(128).half(), torch.zeros(1, 256).half()):
        with pytest.raises(ValueError, match="bias"):
            FPxGatedLinear(64, 128, bias=bias)
    with pytest.raises(ValueError, match="bias"):
        FPxGatedLinear.from_layers(*(FPxLinear(64, 256, bias=torch.zeros(256)) for _ in range(2)))


def test_adapters_that_require_a_gradient_are_refused():
    m, x, index = FPxLinear(64, 256), torch.zeros(2, 64).half(), torch.zeros(2, dtype=torch.int32)
    for name in ("lora_a", "lora_b", "scaling"):
        ad = LowRankAdapters(64, 256, 1, 8)
        getattr(ad, name).requires_grad_()
        with pytest.raises(ValueError, match="no gradient"):
            m(x, ad, index)
        setattr(ad, name, torch.nn.Parameter(getattr(ad, name).detach()))   # (no buffer any more)
        with pytest.raises(ValueError, match="no gradient"):
            m(x, ad, index)


def no_part_of(x):
    """The modules whose kernels have a part in autograd, and calls of theirs on x that a kernel would pass by."""
    mg, ml, ad = FPxGatedLinear(64, 128), FPxLinear(64, 256), LowRankAdapters(64, 256, 1, 8)
    mg, ml, ad = mg.to(x.device), ml.to(x.device), ad.to(x.device)
    ml.input_gradient = True
    index = torch.zeros(x.shape[0], dtype=torch.int32, device=x.device)
    return [lambda t: mg(t), lambda t: ml(t), lambda t: ml(t, ad, index)]


def forward_mode_is_refused(dev):
    fw = torch.autograd.forward_ad
    x, t = torch.ones(3, 64, device=dev).half(), torch.ones(3, 64, device=dev).half()
    for call in no_part_of(x):
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="forward mode"):
                call(fw.make_dual(x, t))
        with pytest.raises(RuntimeError, match="forward mode"):
            torch.func.jvp(call, (x,), (t,))


def test_forward_mode_is_refused():
    forward_mode_is_refused("cpu")


@gpu
def test_forward_mode_is_refused_on_the_gpu():
    forward_mode_is_refused(DEV)
    # where no tangent comes in, the level that is open is nobody's business
    x = torch.ones(3, 64, device=DEV).half()
    for call in no_part_of(x)[:2]:
        want = call(x)
        with torch.autograd.forward_ad.dual_level():
            assert torch.equal(call(x), want)
    # a long prompt with a tangent goes through the library, as it does without input_gradient
    m, x = FPxLinear(64, 256).to(DEV), torch.ones(LONG + 8, 64, device=DEV).half()
    m.input_gradient = True
    with torch.autograd.forward_ad.dual_level():
        assert torch.autograd.forward_ad.unpack_dual(m(torch.autograd.forward_ad.make_dual(x, x))).tangent is not None


def traces_are_refused(dev):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.ones(3, 64, device=dev).half()
    for i, call in enumerate(no_part_of(x)):
        for t in (x, x.clone().requires_grad_()):
            if (i == 1 and not t.requires_grad) or (i == 2 and t.requires_grad):
                continue   # (the layer as it always was; refused anyway)
            with pytest.raises(RuntimeError, match="trace"):
                torch.jit.trace(call, (t,), check_trace=False)
            for pre_dispatch in (False, True):
                with pytest.raises(RuntimeError, match="trace"):
                    make_fx(call, pre_dispatch=pre_dispatch)(t)


def test_traces_are_refused():
    traces_are_refused("cpu")


@gpu
def test_traces_are_refused_on_the_gpu():
    traces_are_refused(DEV)


@gpu
def test_captured_step_with_a_gradient_between_two_boundaries():
    """The copy of such a gradient is part of the graph, and is made anew in every replay."""
    if fp6._ext is None:   # (nothing says there where a gradient would go)
        pytest.skip("a differentiable call is captured with the extension alone")
    mg = block(Weight(2, 2, 2, 512, 320, True))
    weights = randn(2, 1 + 40 * 256, scale=0.1)

    def step(t):
        return torch.autograd.grad(torch.cat([t.flatten()[:1], mg(t).flatten()]), t, weights)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(randn(1, 40, 320).requires_grad_())
        leaf = randn(1, 40, 320).requires_grad_()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            g = step(leaf)
        for seed in range(4):
            weights.copy_(randn(20 + seed, 1 + 40 * 256, scale=0.1))
            with torch.no_grad():
                leaf.copy_(randn(10 + seed, 40, 320))
            want = step(leaf.detach().clone().requires_grad_())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(g, want)


def test_negative_views_are_resolved(monkeypatch):
    """A tensor may say that its values are those in memory with the other sign (the imaginary part of a conjugate does); the kernels read memory."""
    from fp6_llm_amd import module
    seen = []

    def stand_in(E, M, x, *args, **kw):
        seen.append(not x.is_neg() and (x == -1).all())
        return torch.zeros(x.shape[0], 256 if args[2] == 256 else 128, dtype=torch.float16)
    monkeypatch.setattr(module.ops, "gated_forward_native", stand_in)
    monkeypatch.setattr(module.ops, "adapter_forward_native", stand_in)
    x = torch._neg_view(torch.ones(3, 64).half())
    FPxGatedLinear(64, 128)(x)
    FPxLinear(64, 256)(x, LowRankAdapters(64, 256, 1, 8), torch.zeros(3, dtype=torch.int32))
    g = module._gradient(x)
    assert seen == [True, True] and not g.is_neg() and (g == -1).all()
