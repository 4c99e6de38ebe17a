"""Tokens sorted by expert, the experts' rows summed back to tokens, their gradients, and the products of sorted rows, against their definitions in 64 bits.

Tolerances count roundings: half a step of fp16 is 2^-11 of the value (2^-25 below the normal numbers), of bf16 2^-8, of float32 2^-24; a float32 sum of n products is off by at most n * 2^-23
of the sum of their magnitudes, whatever the order."""
import numpy as np
import pytest
import torch

import fp6_llm_amd as fp6
from fp6_llm_amd import _lib
from test_int4 import HALF, TILES, TINY, UNPAIRED, Weight, by_kernel, d, gated64, plain, product64, randn, within

DEV = "cuda:0"
gpu = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def route(seed, T, k, E, drop=0.0, skew=True, dtype=torch.int64):
    """index [T, k] with repeated experts here and there, some of them without a row, -1 and numbers beyond E for a share of the places."""
    rng = np.random.default_rng(seed)
    p = rng.random(E) ** 3 + 1e-3 if skew else np.ones(E)
    index = rng.choice(E, (T, k), p=p / p.sum())
    gone = rng.random((T, k)) < drop
    return torch.from_numpy(np.where(gone, rng.choice([-1, E, E + 5, -7], (T, k)), index)).to(dtype).to(DEV)


class Plan64:
    """The plan from its definition."""

    def __init__(self, index, E):
        e = index.cpu().numpy().reshape(-1)
        e = np.where((e < 0) | (e >= E), E, e)
        self.order = np.argsort(e, kind="stable")
        self.place = np.argsort(self.order, kind="stable")
        self.offsets = np.concatenate(([0], np.cumsum(np.bincount(e, minlength=E + 1)[:E])))
        self.n, self.T, self.k, self.E = self.offsets[-1], *index.shape, E

    def check(self, plan):
        assert (plan.tokens, plan.k, plan.experts, plan.places) == (self.T, self.k, self.E, self.T * self.k)
        assert (plan.offsets.cpu().numpy() == self.offsets).all()
        assert (plan.place.cpu().numpy() == self.place).all()
        assert (plan.order.cpu().numpy() == np.where(np.arange(self.T * self.k) < self.n, self.order, -1)).all()

    def sort(self, x):
        rows = torch.zeros(self.T * self.k, x.shape[1], dtype=x.dtype)
        rows[:self.n] = x.cpu()[torch.from_numpy(self.order[:self.n] // self.k)]
        return rows

    def of_tokens(self, rows):
        """[T, k, H] of sorted rows, and which of them have an expert."""
        place = torch.from_numpy(self.place)
        return rows.cpu()[place].view(self.T, self.k, -1), (place < int(self.n)).view(self.T, self.k, 1)


ROUTES = [  # tokens, k, experts, share without one
    (1, 1, 1, 0.0), (1, 2, 8, 0.0), (1, 8, 64, 0.0), (1, 3, 4, 1.0), (5, 2, 3, 0.3), (16, 4, 64, 0.0), (33, 9, 5, 0.2), (7, 64, 1024, 0.1), (100, 1, 1, 0.0), (257, 7, 100, 0.0), (2048, 1, 16, 0.1), (1024, 2, 8, 0.0),
    (1025, 2, 8, 0.0), (2049, 1, 1, 0.0), (683, 3, 7, 0.5), (4099, 2, 8, 0.05), (1000, 8, 128, 0.0), (333, 64, 1000, 0.1), (5000, 6, 3, 1.0), (40000, 2, 8, 0.0), (30000, 8, 256, 0.02), (70000, 1, 64, 0.0)]


@gpu
@pytest.mark.parametrize("T,k,E,drop", ROUTES)
def test_plan(T, k, E, drop):
    for dtype in (torch.int64, torch.int32):
        index = route(T + k + E, T, k, E, drop, dtype=dtype)
        Plan64(index, E).check(fp6.expert_plan(index, E))


@gpu
@pytest.mark.parametrize("T,k,E,H,drop,type", [(1, 2, 8, 4096, 0.0, "fp16"), (3, 4, 4, 1, 0.2, "bf16"), (16, 4, 64, 2304, 0.0, "fp32"), (65, 2, 8, 333, 0.2, "fp16"), (31, 9, 3, 1001, 0.0, "fp32"), (1, 1, 1, 8, 1.0, "bf16"),
                                                (1030, 2, 8, 520, 0.1, "bf16"), (700, 5, 17, 77, 0.1, "fp16"), (4099, 1, 8, 1030, 0.0, "fp32"), (3001, 8, 128, 64, 0.02, "fp16")])
def test_sort_and_its_gradient(T, k, E, H, drop, type):
    index, dtype = route(T * k + H, T, k, E, drop), TYPES[type]
    x, grad = randn(1, T, H, dtype=dtype).requires_grad_(), randn(2, T * k, H, dtype=dtype)
    want = Plan64(index, E)
    rows, plan = fp6.expert_sort(x, index, E)
    want.check(plan)
    assert rows.dtype == dtype and torch.equal(rows.detach().cpu(), want.sort(x.detach()))
    with torch.no_grad():
        again, plan = fp6.expert_sort(x, index, E)
    want.check(plan)
    assert torch.equal(again, rows)
    dx, = torch.autograd.grad(rows, x, grad)
    g, valid = want.of_tokens(grad.cpu().double())
    g = torch.where(valid, g, 0.0)
    s = g.sum(1)
    within(dx, s, k * 2.0 ** -23 * g.abs().sum(1) + HALF[dtype] * s.abs() + TINY[dtype])


COMBINE = [(1, 8, 64, 8192, 0.0, "fp16", "fp16"), (1, 1, 1, 1, 0.0, "fp32", "fp32"), (5, 3, 4, 7, 0.4, "bf16", "bf16"), (40, 2, 8, 2305, 0.1, "fp32", "fp32"), (33, 9, 16, 2048, 0.0, "fp16", "fp16"), (64, 4, 8, 1024, 0.1, "fp32", "fp16"),
           (17, 5, 8, 999, 0.1, "fp32", "bf16"), (1500, 2, 8, 264, 0.05, "bf16", "bf16"), (3, 64, 100, 40, 0.2, "fp16", "fp16"), (2, 4, 4, 4096, 1.0, "fp16", "fp16")]


@gpu
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,k,E,H,drop,type,to", COMBINE)
def test_combine_and_its_gradients(T, k, E, H, drop, type, to, weighted):
    index, dtype, out_type = route(T * k + H, T, k, E, drop), TYPES[type], TYPES[to]
    rows = randn(1, T * k, H, dtype=dtype).requires_grad_()
    w = torch.rand(T, k, generator=torch.Generator().manual_seed(3)).to(DEV).requires_grad_() if weighted else None
    grad = randn(2, T, H, dtype=out_type)
    plan, want = fp6.expert_plan(index, E), Plan64(index, E)
    y = fp6.expert_combine(rows, plan, w, out_type)
    r, valid = want.of_tokens(d(rows))
    terms = torch.where(valid, r * (d(w)[:, :, None] if weighted else 1.0), 0.0)
    s = terms.sum(1)
    assert y.dtype == out_type
    within(y, s, k * 2.0 ** -23 * terms.abs().sum(1) + HALF[out_type] * s.abs() + TINY[out_type])
    with torch.no_grad():
        assert torch.equal(fp6.expert_combine(rows, plan, w, out_type), y)
    grads = torch.autograd.grad(y, (rows, w) if weighted else (rows,), grad)
    g = d(grad)[:, None]
    back = torch.where(valid, g * (d(w)[:, :, None] if weighted else 1.0), 0.0).flatten(0, 1)
    sorted_back = torch.empty_like(back)
    sorted_back[torch.from_numpy(want.place)] = back
    assert grads[0].dtype == dtype
    within(grads[0], sorted_back, (HALF[dtype] + 2.0 ** -24) * sorted_back.abs() + TINY[dtype], "rows")
    if weighted:
        p = torch.where(valid, g * r, 0.0)
        within(grads[1], p.sum(2), H * 2.0 ** -23 * p.abs().sum(2), "weights")


@gpu
def test_gradients_against_differences():
    """Both are linear in each input, so a central difference is the derivative but for rounding; the loss is a sum of squares over a sort, a nonlinearity and a combine."""
    T, k, E, H = 7, 3, 4, 12
    index = route(5, T, k, E, 0.2)

    def loss(x, w):
        rows, plan = fp6.expert_sort(x, index, E)
        return fp6.expert_combine(rows * rows, plan, w).square().sum()
    x, w = randn(1, T, H, dtype=torch.float32), randn(2, T, k, dtype=torch.float32)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(loss(xg, wg), (xg, wg))
    for seed in range(4):
        dx, dw, h = randn(seed + 10, T, H, dtype=torch.float32), randn(seed + 20, T, k, dtype=torch.float32), 2.0 ** -7
        with torch.no_grad():
            diff = (loss(x + h * dx, w + h * dw) - loss(x - h * dx, w - h * dw)).double() / (2 * h)
            size = (loss(x.abs() + h * dx.abs(), w.abs() + h * dw.abs())).double()
        want = (gx.double() * dx).sum() + (gw.double() * dw).sum()
        # the third derivative's part, h^2 / 6 of a polynomial of degree 6 with terms below `size` (6 * 5 * 4 / 6 = 20 of it), and rounding of the two sums
        assert abs(diff - want) <= 20 * h * h * size + 2.0 ** -16 * size / h


@gpu
def test_numbers_of_rows_without_an_expert_reach_nothing():
    T, k, E, H = 50, 4, 8, 96
    index = route(3, T, k, E, 0.4)
    plan, want = fp6.expert_plan(index, E), Plan64(index, E)
    rows = randn(1, T * k, H)
    rows[int(want.n):] = float("nan")
    w = torch.rand(T, k, device=DEV)
    w[(index < 0) | (index >= E)] = float("inf")
    rows.requires_grad_(), w.requires_grad_()
    y = fp6.expert_combine(rows, plan, w)
    gr, gw = torch.autograd.grad(y, (rows, w), randn(2, T, H))
    assert y.isfinite().all() and gr.isfinite().all() and gw.isfinite().all()
    assert (gr[int(want.n):] == 0).all() and (gw[(index < 0) | (index >= E)] == 0).all()
    x = randn(4, T, H).requires_grad_()
    sorted_rows, _ = fp6.expert_sort(x, index, E)
    g = randn(5, T * k, H)
    g[int(want.n):] = float("nan")
    assert torch.autograd.grad(sorted_rows, x, g)[0].isfinite().all() and (sorted_rows[int(want.n):] == 0).all()


@gpu
def test_a_token_may_name_an_expert_twice():
    index = torch.tensor([[2, 2, 0], [1, 1, 1]], device=DEV)
    x = randn(1, 2, 40, dtype=torch.float32)
    rows, plan = fp6.expert_sort(x, index, 3)
    assert plan.order.tolist() == [2, 3, 4, 5, 0, 1] and plan.offsets.tolist() == [0, 1, 4, 6]
    assert torch.equal(fp6.expert_combine(rows, plan), 3 * x)


@gpu
def test_no_tokens():
    for dtype in (torch.int64, torch.int32):
        index = torch.empty(0, 2, dtype=dtype, device=DEV)
        x = torch.empty(0, 64, dtype=torch.float16, device=DEV, requires_grad=True)
        rows, plan = fp6.expert_sort(x, index, 5)
        assert rows.shape == (0, 64) and plan.offsets.tolist() == [0] * 6 and plan.order.shape == plan.place.shape == (0,)
        y = fp6.expert_combine(rows, plan, torch.empty(0, 2, device=DEV))
        assert y.shape == (0, 64)
        y.sum().backward()
        assert x.grad.shape == (0, 64)
    w = Weight(1, 32, 64, 32, E=5)
    assert fp6.int4_forward_native(rows.detach(), w.native, w.native_scales, plan=plan).shape == (0, 32)


@gpu
def test_strides_views_and_broadcast_gradients():
    T, k, E, H = 37, 3, 5, 72
    index = route(8, T, k, E, 0.1)
    want = Plan64(index, E)
    wide = randn(1, T, 3 * H + 1)
    for x in (wide[:, 1:1 + H], wide[:, H:2 * H], wide.t()[:H].t(), wide[0, :H].expand(T, H), torch.empty(H, T + 1, dtype=torch.float16, device=DEV).normal_().t()[1:], wide.view(-1)[3:3 + T * H].view(T, H)):
        rows, plan = fp6.expert_sort(x, index, E)
        assert torch.equal(rows.cpu(), want.sort(x))
    index2 = torch.stack((index, index), 2)[:, :, 1]   # (a view with strides)
    Plan64(index, E).check(fp6.expert_plan(index2, E))
    rows = randn(2, T * k, 2 * H)[:, 4:4 + H]
    w = torch.rand(T, 2 * k, device=DEV)[:, ::2]
    y = fp6.expert_combine(rows, plan, w)
    assert torch.equal(y, fp6.expert_combine(rows.contiguous(), plan, w.contiguous()))
    # gradients that are broadcast, or begin between two 16-byte boundaries, or are negative views
    rows, w = rows.contiguous().requires_grad_(), w.contiguous().requires_grad_()
    first = torch.autograd.grad(fp6.expert_combine(rows, plan, w).sum(), (rows, w))
    second = torch.autograd.grad(fp6.expert_combine(rows, plan, w), (rows, w), torch.ones(T, H, dtype=torch.float16, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    g = randn(3, T * H + 3)
    third = torch.autograd.grad(fp6.expert_combine(rows, plan, w), (rows, w), g[3:].view(T, H))
    fourth = torch.autograd.grad(fp6.expert_combine(rows, plan, w), (rows, w), g[3:].clone().view(T, H))
    assert torch.equal(third[0], fourth[0])   # (another vector width adds the weights' sums up in another order)
    within(third[1], d(fourth[1]), H * 2.0 ** -23 * (d(g[3:]).view(T, 1, H) * want.of_tokens(d(rows))[0]).abs().sum(2) * 2)
    negative = torch.complex(torch.zeros(T, H, device=DEV), randn(6, T, H, dtype=torch.float32)).conj().imag
    assert negative.is_neg() and torch.equal(fp6.expert_sort(negative, index, E)[0], fp6.expert_sort(negative.clone(), index, E)[0])


@gpu
def test_rows_beyond_32_bit_offsets():
    T, k, E, H = 17000, 4, 8, 32768
    index = route(2, T, k, E, skew=False)
    x = torch.empty(T, H, dtype=torch.float16, device=DEV)
    x[:] = torch.arange(T, device=DEV).remainder(2048).half()[:, None]
    rows, plan = fp6.expert_sort(x, index, E)
    assert rows.numel() > 2 ** 31
    want = (plan.order // k).remainder(2048).half()
    assert torch.equal(rows[:, 0], want) and torch.equal(rows[:, -1], want) and torch.equal(rows[-1], want[-1].expand(H))
    y = fp6.expert_combine(rows, plan, torch.full((T, k), 0.25, device=DEV))
    assert torch.equal(y, x)


@gpu
def test_captured_routing_replays_to_the_eager_results():
    """Index, tokens and weights change between the replays; two graphs and eager calls come in between each other (the larger sort has scratch)."""
    graphs = []
    for T, k, E, H in ((9, 2, 8, 256), (1500, 2, 16, 264)):
        index, x, w = route(1, T, k, E), randn(1, T, H), torch.rand(T, k, device=DEV)
        fp6.expert_combine(fp6.expert_sort(x, index, E)[0], fp6.expert_plan(index, E), w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rows, plan = fp6.expert_sort(x, index, E)
            y = fp6.expert_combine(rows, plan, w)
        graphs.append((graph, index, x, w, rows, plan, y, E))
    for seed in range(2, 6):
        for graph, index, x, w, rows, plan, y, E in graphs:
            index.copy_(route(seed, *index.shape, E, 0.2)), x.copy_(randn(seed, *x.shape)), w.copy_(torch.rand(*w.shape, generator=torch.Generator().manual_seed(seed)))
        eager = [fp6.expert_sort(g[2], g[1], g[-1]) for g in graphs]
        for g in graphs:
            g[0].replay()
        for g in reversed(graphs):
            g[0].replay()
        torch.cuda.synchronize()
        for (graph, index, x, w, rows, plan, y, E), (want, p) in zip(graphs, eager):
            Plan64(index, E).check(plan)
            assert torch.equal(rows, want) and torch.equal(y, fp6.expert_combine(want, p, w))


@gpu
def test_captured_training_step():
    T, k, E, H = 40, 2, 4, 64
    index, x, w = route(1, T, k, E), randn(1, T, H).requires_grad_(), torch.rand(T, k, device=DEV).requires_grad_()

    def step():
        rows, plan = fp6.expert_sort(x, index, E)
        return torch.autograd.grad(fp6.expert_combine(rows * rows, plan, w).float().square().mean(), (x, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(2, 6):
        with torch.no_grad():
            index.copy_(route(seed, T, k, E, 0.1)), x.copy_(randn(seed, T, H))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_a_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    T, k, E, H = 8, 2, 4, 64
    index, x, w = route(1, T, k, E), randn(1, T, H).requires_grad_(), torch.rand(T, k, device=DEV).requires_grad_()
    alive, plan = fp6.expert_sort(x, index, E)
    kept = fp6.expert_combine(alive.detach(), plan, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            fp6.expert_sort(x, index, E)
        with pytest.raises(RuntimeError):
            fp6.expert_combine(alive.detach(), plan, w)
        out = alive.detach() + 1
    del kept
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive.detach() + 1)


@gpu
@pytest.mark.parametrize("T", [6, 1400])
def test_calls_without_the_extension(T, monkeypatch):
    assert fp6._ext is not None
    k, E, H = 3, 8, 136
    index, x, w = route(1, T, k, E, 0.1), randn(1, T, H).requires_grad_(), torch.rand(T, k, device=DEV).requires_grad_()
    g, wide = randn(2, T, H), randn(3, T * k, H, dtype=torch.float32)
    weights = Weight(2, 64, 136 // 32 * 32, 32, True, E=E)

    def all_of():
        rows, plan = fp6.expert_sort(x, index, E)
        y = fp6.expert_combine(rows, plan, w)
        grads = torch.autograd.grad(y, (x, w), g)
        product = fp6.int4_forward_native(rows.detach()[:, :128].contiguous(), weights.native, weights.native_scales, plan=plan)
        return [rows, plan.table, y, *grads, fp6.expert_combine(wide, plan, None, torch.bfloat16), product]
    first = all_of()
    monkeypatch.setattr(fp6, "_ext", None)
    for a, b in zip(first, all_of()):
        assert a.dtype == b.dtype and torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------- products of sorted rows
GROUPED = [  # tokens, k, experts, OC, IC, group, zeros, type, share without an expert, activation, bias
    (1, 2, 8, 256, 512, 128, False, "fp16", 0.0, None, False), (1, 1, 3, 32, 32, 32, True, "bf16", 0.0, "silu", True), (1, 4, 4, 48, 160, 64, True, "fp16", 1.0, None, True), (9, 2, 3, 96, 480, 32, True, "fp16", 0.2, "gelu", True),
    (40, 8, 64, 288, 608, 64, True, "bf16", 0.0, "silu", False), (60, 2, 100, 64, 256, 128, False, "fp16", 0.1, None, True), (33, 3, 2, 272, 352, 32, False, "bf16", 0.3, None, False), (150, 2, 4, 544, 416, 64, True, "fp16", 0.1, "gelu_tanh", True),
    (300, 1, 5, 1056, 160, 128, True, "bf16", 0.2, "silu", True), (700, 2, 8, 288, 544, 32, True, "fp16", 0.05, "silu", False), (513, 1, 1, 96, 256, 128, False, "fp16", 0.0, None, False), (64, 8, 256, 32, 64, 64, False, "bf16", 0.0, None, False),
    (1100, 4, 16, 160, 736, 96, True, "bf16", 0.0, "gelu", True)]


def grouped64(w, plan, rows, bias, act, dtype):
    """Want and tolerance of the product of sorted rows; those behind the last are zeros."""
    want, tol = [], []
    for e in range(plan.E):
        lo, hi = int(plan.offsets[e]), int(plan.offsets[e + 1])
        y, err = product64(w.w[e], rows[lo:hi], None if bias is None else bias[e])
        y, t = plain(y, err, dtype) if act is None else gated64(y, err, act, dtype)
        want.append(y), tol.append(t)
    rest = torch.zeros(plan.T * plan.k - int(plan.n), want[0].shape[1], dtype=torch.float64)
    return torch.cat(want + [rest]), torch.cat(tol + [rest])


@gpu
@pytest.mark.parametrize("T,k,E,OC,IC,group,zeros,type,drop,act,bias", GROUPED)
def test_product_of_sorted_rows(T, k, E, OC, IC, group, zeros, type, drop, act, bias):
    w, index = Weight(T + OC + IC, OC, IC, group, zeros, type, E), route(T + E, T, k, E, drop)
    x, b = randn(T, T, IC, dtype=w.dtype), randn(1, E, OC, dtype=w.dtype) if bias else None
    rows, plan = fp6.expert_sort(x, index, E)
    want, tol = grouped64(w, Plan64(index, E), rows, b, act, w.dtype)
    out = torch.full_like(want, float("nan"), dtype=w.dtype, device=DEV)
    within(fp6.int4_forward_native(rows, w.native, w.native_scales, plan=plan, activation=act, bias=b, out=out), want, tol)
    if act is None:
        got = fp6.int4_forward_native(rows, w.native, w.native_scales, plan=plan, bias=b, out_dtype=torch.float32)
        within(got, *grouped64(w, Plan64(index, E), rows, b, act, torch.float32), "float32")


@gpu
@pytest.mark.parametrize("sizes", [[0, 0, 5, 0], [16, 17, 0, 1], [64, 0, 65, 63, 1, 128], [1] * 70, [0] * 130 + [3], [300, 0, 1], [129, 127, 128]])
def test_experts_with_these_many_rows(sizes):
    """Borders of experts inside, at and behind the kernels' tiles; behind the last expert rows without one."""
    E, rest = len(sizes), 7
    index = torch.tensor([e for e, n in enumerate(sizes) for _ in range(n)] + [-1] * rest).unsqueeze(1)
    index = index[torch.randperm(len(index), generator=torch.Generator().manual_seed(1))].to(DEV)
    w = Weight(E, 80, 288, 32, True, "fp16", E)
    rows, plan = fp6.expert_sort(randn(2, len(index), 288), index, E)
    within(fp6.int4_forward_native(rows, w.native, w.native_scales, plan=plan), *grouped64(w, Plan64(index, E), rows, None, None, torch.float16))


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_c_abi():
    L, p = _lib.lib(), 1 << 20   # (an address that nothing reads: every call is refused before a launch)
    SHAPE, NULL, WORKSPACE, ALIGN, TYPE = -2, -3, -4, -6, -10

    def sort(index=p, wide=1, offsets=p, order=p, place=p, x=p, ldx=64, rows=p, T=4, k=2, E=8, H=64, dtype=0, ws=None):
        return L.fp6mi_expert_sort(None, index, wide, offsets, order, place, x, ldx, rows, T, k, E, H, dtype, ws)
    for bad in (dict(k=0), dict(k=65), dict(E=0), dict(E=1025), dict(T=1 << 30), dict(H=0), dict(ldx=63), dict(H=(1 << 24) + 1, ldx=1 << 25)):
        assert sort(**bad) == SHAPE, bad
    for name in ("index", "offsets", "order", "place", "x"):
        assert sort(**{name: None}) == NULL, name
    for bad in (dict(index=p + 4), dict(index=p + 2, wide=0), dict(offsets=p + 2), dict(order=p + 1), dict(place=p + 2), dict(x=p + 1), dict(rows=p + 2, dtype=2), dict(T=4000, ws=p + 8)):
        assert sort(**bad) == ALIGN, bad
    assert sort(dtype=3) == TYPE and sort(dtype=-1) == TYPE and sort(T=4000) == WORKSPACE
    assert L.fp6mi_expert_sort_workspace_bytes(4, 2, 8) == 0 and L.fp6mi_expert_sort_workspace_bytes(4000, 2, 8) > 0 and L.fp6mi_expert_sort_workspace_bytes(4000, 0, 8) == 0

    def combine(rows=p, place=p, valid=p, weights=p, out=p, T=4, k=2, H=64, r=0, o=0):
        return L.fp6mi_expert_combine(None, rows, place, valid, weights, out, T, k, H, r, o)
    for bad in (dict(k=0), dict(k=65), dict(H=0), dict(H=(1 << 24) + 1), dict(T=1 << 30)):
        assert combine(**bad) == SHAPE, bad
    for r, o in ((0, 1), (1, 0), (0, 2), (3, 3), (2, 3), (-1, 0)):
        assert combine(r=r, o=o) == TYPE
    for name in ("rows", "place", "valid", "out"):
        assert combine(**{name: None}) == NULL, name
    for name, by in (("rows", 1), ("place", 2), ("valid", 2), ("weights", 2), ("out", 1)):
        assert combine(**{name: p + by}) == ALIGN, name
    assert combine(T=0) == 0

    def backward(grad=p, rows=p, place=p, valid=p, weights=p, gr=p, gw=p, T=4, k=2, H=64, r=0, o=0):
        return L.fp6mi_expert_combine_backward(None, grad, rows, place, valid, weights, gr, gw, T, k, H, r, o)
    assert backward(k=0) == SHAPE and backward(r=1, o=0) == TYPE and backward(T=0) == 0
    for bad in (dict(grad=None), dict(place=None), dict(valid=None), dict(rows=None), dict(gr=None, gw=None)):
        assert backward(**bad) == NULL, bad
    for name, by in (("grad", 1), ("rows", 1), ("place", 2), ("valid", 2), ("weights", 2), ("gr", 1), ("gw", 2)):
        assert backward(**{name: p + by}) == ALIGN, name


def refusals(dev, monkeypatch):
    index, x = torch.zeros(4, 2, dtype=torch.int64, device=dev), torch.zeros(4, 64, dtype=torch.float16, device=dev)
    plan = fp6.experts.ExpertPlan(torch.zeros(20, dtype=torch.int32, device=dev), 4, 2, 3)
    short = fp6.experts.ExpertPlan(torch.zeros(19, dtype=torch.int32, device=dev), 4, 2, 3)
    rows, weights = torch.zeros(8, 64, dtype=torch.float16, device=dev), torch.zeros(4, 2, device=dev)
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        for bad in (dict(index=index.float()), dict(index=index[0]), dict(index=index[:, :0]), dict(index=index[:, :1].expand(4, 65)), dict(experts=0), dict(experts=1025), dict(x=x[:3]), dict(x=x[0]), dict(x=x.double()),
                    dict(x=x.int()), dict(x=x[:, :0]), dict(index=index.cpu()), dict(x=x.cpu() if dev != "cpu" else x)):
            with pytest.raises(ValueError):
                fp6.expert_sort(**{**dict(x=x, index=index, experts=3), **bad})
        for bad in (dict(rows=rows[:7]), dict(rows=rows[0]), dict(rows=rows.double()), dict(rows=rows.int()), dict(plan=short), dict(dtype=torch.float32), dict(dtype=torch.bfloat16), dict(dtype=torch.float64), dict(weights=weights[:3]),
                    dict(weights=weights[:, :1]), dict(weights=weights.int()), dict(rows=rows.cpu() if dev != "cpu" else rows[:7]), dict(weights=weights.cpu() if dev != "cpu" else weights[:3])):
            for grad in (False, True):
                args = {**dict(rows=rows, plan=plan, weights=weights), **bad}
                if grad and args["rows"].is_floating_point():
                    args["rows"] = args["rows"].detach().clone().requires_grad_()
                with pytest.raises(ValueError):
                    fp6.expert_combine(**args)


def test_refusals_of_the_functions(monkeypatch):
    refusals("cpu", monkeypatch)


@gpu
def test_refusals_of_the_functions_on_the_gpu(monkeypatch):
    refusals(DEV, monkeypatch)


@gpu
def test_forward_mode_transforms_and_traces_are_refused():
    index, x = torch.zeros(4, 2, dtype=torch.int64, device=DEV), randn(1, 4, 64)
    rows, plan = fp6.expert_sort(x, index, 3)
    for f, t in ((lambda t: fp6.expert_sort(t, index, 3)[0], x), (lambda t: fp6.expert_combine(t, plan), rows)):
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
            f(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(t.unsqueeze(0))
        with pytest.raises(RuntimeError):
            torch.jit.trace(f, t)


def test_objects_of_the_makefile_depend_on_all_that_they_include():
    import os
    import re
    from test_build_sources import PACKAGE, included
    with open(os.path.join(PACKAGE, "Makefile")) as f:
        text = f.read()
    headers = re.search(r"^HDRS = (.*)$", text, re.M).group(1)
    rules = re.findall(r"^\$\(OBJ2\)/(\S+)\.o: (.*)$", text, re.M)
    assert {target for target, _ in rules} == {"fp6mi_int4_%", "fp6mi_int4_api", "fp6mi_experts"}
    for target, needs in rules:
        needs = [os.path.normpath(os.path.join(PACKAGE, n)) for n in needs.replace("$(HDRS)", headers).split()]
        missing = included(needs[0]) - set(needs)
        assert not missing, "%s.o: %s" % (target, sorted(os.path.basename(m) for m in missing))


@gpu
def test_second_derivatives_are_refused(monkeypatch):
    T, k, E, H = 5, 2, 3, 16
    index = route(1, T, k, E)
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        x, w = randn(1, T, H, dtype=torch.float32).requires_grad_(), torch.rand(T, k, device=DEV).requires_grad_()
        rows, plan = fp6.expert_sort(x, index, E)
        for y, leaves in ((rows.square().sum(), (x,)), (fp6.expert_combine(rows, plan, w).square().sum(), (x, w))):
            for g in torch.autograd.grad(y, leaves, create_graph=True):
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(g.sum(), x, retain_graph=True)


@gpu
def test_gradients_that_are_not_asked_for():
    T, k, E, H = 6, 2, 3, 40
    index, rows = route(1, T, k, E), randn(1, T * k, H)
    plan, w = fp6.expert_plan(index, E), torch.rand(T, k, device=DEV)
    both_r, both_w = rows.clone().requires_grad_(), w.clone().requires_grad_()
    g = randn(2, T, H)
    want = torch.autograd.grad(fp6.expert_combine(both_r, plan, both_w), (both_r, both_w), g)
    r = rows.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fp6.expert_combine(r, plan, w), r, g)[0], want[0])
    v = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fp6.expert_combine(rows, plan, v), v, g)[0], want[1])
    half = w.double().requires_grad_()   # (weights of another type are converted, and so is their gradient)
    got, = torch.autograd.grad(fp6.expert_combine(rows, plan, half), half, g)
    assert got.dtype == torch.float64 and torch.equal(got.float(), want[1])
    with torch.no_grad():
        assert not fp6.expert_combine(both_r, plan, both_w).requires_grad


@gpu
@pytest.mark.parametrize("kernel", range(12))
@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_every_kernel_with_rows_of_experts(kernel, type):
    """Borders of experts inside tiles, experts without rows, rows behind the last expert's that hold NaN."""
    E, sizes = 5, [3, 0, 40, 17, 129]
    index = torch.tensor([e for e, n in enumerate(sizes) for _ in range(n)] + [-1] * 20).unsqueeze(1).to(DEV)
    w = Weight(kernel, 96, 416, 128 if kernel == 10 else 64, True, type, E)
    rows, plan = fp6.expert_sort(randn(2, len(index), 416, dtype=w.dtype), index, E)
    want = Plan64(index, E)
    b = randn(3, E, 96, dtype=w.dtype)
    y, tol = grouped64(w, want, rows, b, None, w.dtype)
    h, htol = grouped64(w, want, rows, b, "silu", w.dtype)
    extra = 30 if type == "bf16" and kernel not in TILES else 1   # (128 + q and -(128 + z), 143 at most, stand for a difference that is 5 in the mean)
    rows[int(want.n):] = float("nan")
    within(by_kernel(kernel, w, rows, b, plan=plan), y, tol * extra)
    if kernel not in UNPAIRED:
        within(by_kernel(kernel, w, rows, b, act=0, plan=plan), h, htol * extra)


@gpu
def test_weights_beyond_32_bit_offsets():
    """The last of many experts, six gigabytes in, against the same matrix by itself."""
    E, OC, IC = 32, 16384, 24576
    codes = torch.empty(E, OC, IC // 2, dtype=torch.uint8, device=DEV)
    for e in range(E):
        codes[e] = torch.randint(0, 256, (OC, IC // 2), dtype=torch.uint8, device=DEV)
    scales = torch.rand(E, OC, IC // 128, device=DEV).half() / 100
    native, native_scales = fp6.int4_pack_native(codes, scales)
    one, one_scales = fp6.int4_pack_native(codes[E - 1], scales[E - 1])
    assert native.numel() * 4 > 2 ** 32 and torch.equal(native[E - 1], one) and torch.equal(native_scales[E - 1], one_scales)
    for T in (3, 70):
        x, index = randn(1, T, IC), torch.full((T, 1), E - 1, device=DEV)
        rows, plan = fp6.expert_sort(x, index, E)
        k = 4 if T == 3 else 11
        both = Weight.__new__(Weight)
        both.native, both.native_scales, both.OC, both.IC, both.E, both.dtype = native, native_scales, OC, IC, E, torch.float16
        alone = Weight.__new__(Weight)
        alone.native, alone.native_scales, alone.OC, alone.IC, alone.E, alone.dtype = one, one_scales, OC, IC, 0, torch.float16
        assert torch.equal(by_kernel(k, both, rows, plan=plan), by_kernel(k, alone, x))


@gpu
def test_two_threads_on_one_stream():
    """Calls with scratch (many places; bf16 tiles) from two threads: each has the results of its own."""
    import threading
    E, k, T, H = 8, 2, 2000, 256
    w = Weight(1, 512, H, 64, True, "bf16")
    inputs = [(route(s, T, k, E), randn(s, T, H, dtype=torch.bfloat16)) for s in (1, 2)]
    want = [(fp6.expert_sort(x, i, E)[0], fp6.int4_forward_native(x, w.native, w.native_scales)) for i, x in inputs]
    failed = []

    def work(n):
        i, x = inputs[n]
        for _ in range(30):
            rows, y = fp6.expert_sort(x, i, E)[0], fp6.int4_forward_native(x, w.native, w.native_scales)
            if not (torch.equal(rows, want[n][0]) and torch.equal(y, want[n][1])):
                failed.append(n)
    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
