"""The operators around the linear layer (gated feed-forward block, input gradient, low-rank adapters) against their formulas in 64 bits.

Tolerances count roundings: half a step of fp16 is 2^-11 of the value (2^-25 below the normal numbers); a float32 sum of n products, which are exact, is off by at most
n * 2^-23 of the sum of their magnitudes, whatever the order and however the matrix unit rounds between them."""
import numpy as np
import pytest
import torch

import fp6_llm_amd as fp6
from fp6_llm_amd import _lib, quant

FORMATS = [(3, 2), (2, 2), (2, 3), (2, 1)]
ACTS = ["silu", "gelu", "gelu_tanh"]
DEV = "cuda:0"
gpu = pytest.mark.gpu
HALF, TINY = 2.0 ** -11, 2.0 ** -25


def sum_error(n):
    return n * 2.0 ** -23


class Weight:
    """Random codes of a format, row scales and (groups) exponents: on the GPU in the native layout, and as numbers in 64 bits."""

    def __init__(self, seed, E, M, OC, IC, groups=False, pairs=False):
        rng = np.random.default_rng(seed)
        codes = rng.integers(0, 1 << (1 + E + M), (OC, IC)).astype(np.uint8)
        mags = quant.magnitudes(E, M)
        value = mags[codes & ((1 << (E + M)) - 1)] * np.where(codes >> (E + M), -1.0, 1.0)
        scales = (np.exp(0.3 * rng.standard_normal(OC)) / (np.sqrt((mags ** 2).mean()) * np.sqrt(IC))).astype(np.float16)
        exps = rng.integers(122, 129, (OC, (IC + 127) // 128)).astype(np.uint8) if groups else None
        if groups:
            value = value * np.repeat(2.0 ** (exps.astype(np.int64) - 127), 128, axis=1)[:, :IC]
        w = value * scales.astype(np.float64)[:, None]
        self.E, self.M, self.OC, self.IC = E, M, OC, IC
        self.native = fp6.weight_prepacking_native_cpu(E, M, torch.from_numpy(quant.pack_raw(codes, E, M))).to(DEV)
        self.scales = torch.from_numpy(scales).to(DEV)
        self.exps = fp6.pack_group_exps(torch.from_numpy(exps), OC, IC).to(DEV) if groups else None
        self.w = torch.from_numpy(w)

    @property
    def fmt(self):
        return self.E, self.M


def randn(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).half().to(DEV)


def d(t):
    return t.detach().cpu().double()


def within(got, want, tol, what=""):
    got = d(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    bad &= ~(torch.isinf(want) & (got == want))
    assert not bad.any(), "%s: %d of %d off, first at %s: got %s, want %s +- %s" % (
        what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), tol.expand_as(want)[bad][0].item())


def halves(p):
    p = p.reshape(p.shape[0], -1, 2, 16)
    return p[:, :, 0].flatten(1), p[:, :, 1].flatten(1)


def pairs(g, u):
    return torch.stack((g.reshape(g.shape[0], -1, 16), u.reshape(u.shape[0], -1, 16)), 2).flatten(1)


def act64(act, g):
    if act == "silu":
        return g * torch.sigmoid(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")


def slope64(act, g):
    g = g.clone().requires_grad_()
    return torch.autograd.grad(act64(act, g).sum(), g)[0]


def preacts(w, x, bias):
    """Pre-activations in 64 bits and how far float32 sums may be from them."""
    y, mag = d(x) @ w.w.t(), d(x).abs() @ w.w.abs().t()
    if bias is not None:
        y, mag = y + d(bias), mag + d(bias).abs()
    return y, sum_error(w.IC + 1) * mag


# The largest slopes are 1.1 (silu) and 1.13 (gelu); the functions themselves are taken to 2^-18 of |g| at most, which is what 32-bit exponentials of arguments
# up to about 2^4 and error functions give.
def gated64(w, x, bias, act):
    y, err = preacts(w, x, bias)
    (g, u), (eg, eu) = halves(y), halves(err)
    a = act64(act, g)
    ea = 1.13 * eg + 2.0 ** -18 * g.abs()
    h = a * u
    return y, err, h, (ea * u.abs() + eu * a.abs() + ea * eu) * (1 + HALF) + HALF * h.abs() + TINY


GATED = [  # E, M, OC, IC, N, activation, group exponents, bias
    (3, 2, 256, 64, 1, "silu", False, False), (2, 2, 512, 320, 2, "gelu", True, True), (2, 1, 256, 1024, 7, "gelu_tanh", False, True), (2, 3, 768, 576, 9, "silu", True, False),
    (3, 2, 1024, 512, 16, "gelu", False, True), (3, 2, 512, 256, 17, "silu", True, True), (2, 2, 1280, 832, 33, "silu", False, False), (2, 1, 512, 1088, 48, "gelu", True, False),
    (2, 3, 2304, 448, 65, "gelu_tanh", False, True), (3, 2, 512, 2048, 97, "silu", True, False), (2, 2, 1536, 704, 130, "silu", True, True), (3, 2, 2560, 640, 300, "gelu", False, False),
    (2, 1, 768, 512, 515, "silu", False, True), (2, 3, 3328, 1216, 777, "gelu_tanh", True, True), (3, 2, 4608, 4544, 40, "silu", False, False), (3, 2, 22016, 1024, 1, "silu", False, True),
    (2, 1, 256, 8192, 5, "silu", False, False), (3, 2, 256, 8192, 200, "silu", False, True), (3, 2, 8192, 512, 1100, "silu", False, True)]


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,act,groups,bias", GATED)
def test_gated_block_forward(E, M, OC, IC, N, act, groups, bias):
    w = Weight(OC + IC + N, E, M, OC, IC, groups)
    x, b = randn(N, N, IC), randn(N + 1, OC, scale=0.3) if bias else None
    y, err, h, tol = gated64(w, x, b, act)
    got = fp6.gated_forward_native(E, M, x, w.native, w.scales, OC, act, group_exps=w.exps, bias=b)
    within(got, h, tol, "out")
    pre = torch.full((N, OC), float("nan"), device=DEV)
    again = fp6.gated_forward_native(E, M, x, w.native, w.scales, OC, act, preact=pre, group_exps=w.exps, bias=b)
    within(again, h, tol, "out beside preact")
    within(pre, y, err, "preact")


@gpu
@pytest.mark.parametrize("splitK", [2, 3, 8])
@pytest.mark.parametrize("N", [3, 50, 260])
def test_gated_block_with_k_split(splitK, N):
    w = Weight(splitK, 2, 2, 512, 1344, True)
    x, b = randn(1, N, 1344), randn(2, 512)
    y, err, h, tol = gated64(w, x, b, "silu")
    pre = torch.full((N, 512), float("nan"), device=DEV)
    within(fp6.gated_forward_native(2, 2, x, w.native, w.scales, 512, splitK=splitK, preact=pre, group_exps=w.exps, bias=b), h, tol)
    within(pre, y, err)


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("N,OC,IC", [(1, 256, 64), (37, 512, 320), (200, 768, 1024)])
def test_gated_block_backward(act, N, OC, IC):
    w = Weight(7, 3, 2, OC, IC, True)
    dh, pre = randn(3, N, OC // 2, scale=0.1), randn(4, N, OC, scale=3.0).float() * 1.0001
    pre[0, :16] = torch.tensor([0, -0.0, 1e-7, -1e-7, 12, -12, 60, -60, 300, -300, 2e4, -2e4, 1e9, -1e9, 0.5, -0.5])
    pre[0, 16:32] = 1e-3   # (their slopes, not their size, are looked at)
    dx, dp = fp6.gated_backward_native(3, 2, dh, pre, w.native, w.scales, IC, act, group_exps=w.exps)
    (g, u), dd = halves(d(pre)), d(dh)
    a, s = act64(act, g), slope64(act, g)
    want = pairs(dd * u * s, dd * a)
    # the slope is a sum of terms up to 1.2 + |g| at the most, each to 2^-18; so is the activation
    slack = 2.0 ** -18 * pairs(dd.abs() * u.abs() * (1 + g.abs().clamp(max=12)), dd.abs() * g.abs())
    fits = want.abs() < 65000
    assert (~fits).sum() <= 2 and torch.isinf(d(dp)[~fits]).all()
    within(torch.where(fits, d(dp), want), want, HALF * want.abs() + slack + TINY, "grad_preact")
    assert fits[1:].all()
    # rows behind the first: its products with the weights, from products with the scales' mantissas that were rounded once
    dx64, mag = want[1:] @ w.w, want[1:].abs() @ w.w.abs()
    within(dx[1:], dx64, (sum_error(OC) + HALF) * mag + (slack[1:] + TINY) @ w.w.abs() + HALF * dx64.abs() + TINY, "grad_in")
    dx2, none = fp6.gated_backward_native(3, 2, dh, pre, w.native, w.scales, IC, act, group_exps=w.exps, grad_preact=False)
    assert none is None and torch.equal(dx2[1:], dx[1:])


@gpu
@pytest.mark.parametrize("splitK", [1, 2, 5, 16])
@pytest.mark.parametrize("N", [16, 24, 32, 90])
def test_gated_block_backward_with_the_sum_split(N, splitK):
    """(the kernels for few rows take more wavefronts where a split has many weight rows)"""
    w = Weight(8, 2, 1, 1024, 320, True)
    dh, pre = randn(3, N, 512, scale=0.1), randn(4, N, 1024).float()
    dx, dp = fp6.gated_backward_native(2, 1, dh, pre, w.native, w.scales, 320, splitK=splitK, group_exps=w.exps)
    want, mag = d(dp) @ w.w, d(dp).abs() @ w.w.abs()   # (dp has been rounded once, and what was multiplied once)
    within(dx, want, (sum_error(1024) + 2 * HALF * (1 + HALF)) * mag + 2 * TINY * w.w.abs().sum(0) + HALF * want.abs() + TINY)


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gated_block_gradient_against_differences(act):
    """The whole chain: the slope of sum(dh * h) along a direction, from the kernels' gradient and from central differences of the formula in 64 bits."""
    N, OC, IC = 19, 512, 448
    w = Weight(11, 2, 3, OC, IC)
    x, dh = randn(5, N, IC), randn(6, N, OC // 2)
    pre = torch.empty(N, OC, device=DEV)
    fp6.gated_forward_native(2, 3, x, w.native, w.scales, OC, act, preact=pre)
    dx, dp = fp6.gated_backward_native(2, 3, dh, pre, w.native, w.scales, IC, act)
    v = torch.randn(N, IC, generator=torch.Generator().manual_seed(8), dtype=torch.float64)

    def f(t):
        g, u = halves((d(x) + t * v) @ w.w.t())
        return (d(dh) * act64(act, g) * u).sum()
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    # Roundings on the way: dx itself, each product of a dp with its mantissa, float32 sums of the pre-activations (second derivatives of the activations are below 1.3) and of dx,
    # activations and slopes to 2^-17
    (g, u), (eg, eu) = halves(d(x) @ w.w.t()), halves(sum_error(IC) * (d(x).abs() @ w.w.abs().t()))
    dd = d(dh).abs()
    ep = pairs(dd * (1.3 * eg * u.abs() + 1.13 * eu + 2.0 ** -17 * u.abs()), dd * (1.13 * eg + 2.0 ** -17 * g.abs())) + (HALF + sum_error(OC)) * d(dp).abs()
    tol = (v.abs() * (HALF * d(dx).abs() + ep @ w.w.abs())).sum()
    assert abs((d(dx) * v).sum() - slope) <= tol
    assert tol < 0.2 * (d(dx) * v).abs().sum()   # (the bound says something)


GRAD = [(3, 2, 256, 64, 1, False), (2, 2, 512, 320, 3, True), (2, 1, 256, 1024, 8, False), (2, 3, 768, 576, 16, True), (3, 2, 1024, 512, 17, False), (2, 2, 256, 192, 32, False),
        (2, 1, 1280, 256, 33, True), (3, 2, 512, 704, 64, True), (2, 3, 512, 1216, 65, False), (2, 2, 2304, 448, 128, True), (3, 2, 768, 832, 129, False), (2, 1, 512, 512, 257, True),
        (2, 3, 1536, 320, 333, True), (3, 2, 4096, 256, 20, False), (3, 2, 8192, 128, 70, False), (3, 2, 256, 4544, 700, False), (2, 2, 768, 2304, 1030, True), (3, 2, 512, 8192, 500, False), (2, 1, 512, 6144, 4000, True), (2, 3, 256, 8192, 1500, True)]


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,groups", GRAD)
def test_input_gradient(E, M, OC, IC, N, groups):
    w = Weight(OC + IC + N, E, M, OC, IC, groups)
    dy = randn(N, N, OC, scale=0.05)
    want, mag = d(dy) @ w.w, d(dy).abs() @ w.w.abs()   # (each product of a dy with the mantissa of its row's scale is rounded once)
    for splits in (None, 1, 3):
        got = fp6.linear_input_grad_native(E, M, dy, w.native, w.scales, IC, splitK=splits, group_exps=w.exps)
        within(got, want, (sum_error(OC + 3) + HALF) * mag + TINY * w.w.abs().sum(0) + HALF * want.abs() + TINY, "splits %s" % splits)


@gpu
def test_input_gradient_keeps_rows_apart():
    """An infinity or a NaN in one batch row touches no other row, and rows behind the last one stay as they were."""
    w = Weight(1, 3, 2, 512, 320)
    for N in (5, 40, 100, 200):
        dy = randn(2, N, 512)
        clean = fp6.linear_input_grad_native(3, 2, dy, w.native, w.scales, 320)
        dy[1, 7], dy[N - 1, 100] = float("inf"), float("nan")
        buf = torch.full((N + 3, 320), 7.0, dtype=torch.float16, device=DEV)
        got = fp6.linear_input_grad_native(3, 2, dy, w.native, w.scales, 320, out=buf[:N])
        keep = [n for n in range(N) if n not in (1, N - 1)]
        assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[N - 1]).all() and (buf[N:] == 7.0).all()
        assert not torch.isfinite(got[1]).any()


@gpu
@pytest.mark.parametrize("E,M", FORMATS)
def test_input_gradient_with_scales_of_every_kind(E, M):
    """Negative, zero, subnormal and large scales, with group exponents: the scale's mantissa goes to dy, its power of two to the weight, which keeps its value as far as fp16 reaches.  (The
    weights of a row with a subnormal scale are rounded to fp16, one rounding more.)"""
    OC, IC, N = 256, 256, 33
    w = Weight(2, E, M, OC, IC, True)
    sc = torch.ones(OC, dtype=torch.float64)
    special = [0.0, -0.0, -1.0, 2.0 ** -24, 3 * 2.0 ** -24, 2.0 ** -14, -1.999 * 2.0 ** -9, 1000.0, -60.0]
    sc[:len(special)] = torch.tensor(special, dtype=torch.float64)
    sc = sc.half().double()
    value = w.w / d(w.scales)[:, None]
    mats = value * sc[:, None]
    power = torch.exp2(torch.floor(torch.log2(sc.abs().clamp(min=2.0 ** -24))))[:, None]
    dy = randn(3, N, OC, scale=2.0 ** -6)
    want, mag = d(dy) @ mats, d(dy).abs() @ mats.abs()
    lost = (d(dy).abs() * (sc.abs() / power[:, 0])) @ torch.full((OC, IC), TINY, dtype=torch.float64)
    got = fp6.linear_input_grad_native(E, M, dy, w.native, sc.half().to(DEV), IC, group_exps=w.exps)
    within(got, want, (sum_error(OC) + 2 * HALF) * mag + lost + TINY * (mats / sc.clamp(min=1e-9)[:, None]).abs().nan_to_num().sum(0) + HALF * want.abs() + TINY)


@gpu
@pytest.mark.parametrize("N", [5, 40, 200])
def test_scales_that_start_between_two_16_byte_boundaries(N):
    """(scales and bias are halfs, and may start at any of them)"""
    w = Weight(3, 3, 2, 512, 320)
    odd, b = torch.empty(513, dtype=torch.float16, device=DEV)[1:].copy_(w.scales), torch.empty(513, dtype=torch.float16, device=DEV)[1:].copy_(randn(9, 512))
    x, dy, dh = randn(1, N, 320), randn(2, N, 512), randn(3, N, 256)
    pres, outs = [torch.empty(N, 512, device=DEV) for _ in range(2)], []
    ad = (*bank(3, 3, 16, 512, 320), (torch.arange(N, device=DEV) % 4 - 1).int())
    for sc, bias, pre in ((w.scales, b.clone(), pres[0]), (odd, b, pres[1])):
        assert sc.is_contiguous() and sc.data_ptr() % 16 == (2 if sc is odd else 0)
        outs.append([fp6.gated_forward_native(3, 2, x, w.native, sc, 512, preact=pre, bias=bias), pre, *fp6.gated_backward_native(3, 2, dh, pre, w.native, sc, 320),
                     fp6.linear_input_grad_native(3, 2, dy, w.native, sc, 320), fp6.adapter_forward_native(3, 2, x, w.native, sc, 512, *ad, bias=bias)])
    assert all(torch.equal(p, q) for p, q in zip(*outs))


@gpu
@pytest.mark.parametrize("N", [3, 30, 100])
def test_gradients_up_to_the_largest_half(N):
    """Scaled losses make gradients of any size: up to 65504 they go in as they are, whatever the mantissas of the scales, and what comes out of small weights is finite."""
    OC, IC = 512, 320
    w = Weight(4, 3, 2, OC, IC)
    sc = (torch.linspace(1.0, 1.999, OC, dtype=torch.float64) * 2.0 ** -13).half()
    mats = w.w / d(w.scales)[:, None] * sc.double()[:, None]
    g = torch.Generator().manual_seed(N)
    dy = ((40000 + 25504 * torch.rand(N, OC, generator=g)) * (2 * torch.randint(0, 2, (N, OC), generator=g) - 1)).half().to(DEV)
    dy[0, :2] = torch.tensor([65504.0, -65504.0])
    want, mag = d(dy) @ mats, d(dy).abs() @ mats.abs()
    assert want.abs().max() < 65504
    got = fp6.linear_input_grad_native(3, 2, dy, w.native, sc.to(DEV), IC)
    # (weights of small scales may lose bits below the normal halfs: 2^-25, against scales of 2^-13)
    within(got, want, (sum_error(OC) + HALF) * mag + 2 * TINY * d(dy).abs().sum(1, keepdim=True) + HALF * want.abs() + TINY)
    # and through the block: g = 0 has slope 1/2 and activation 0, so dp = dh * u / 2 there
    pre = torch.zeros(N, OC, device=DEV)
    pre.view(N, -1, 2, 16)[:, :, 1] = 2.0
    dh = dy[:, :OC // 2]
    dx, dp = fp6.gated_backward_native(3, 2, dh, pre, w.native, sc.to(DEV), IC)
    dp64 = pairs(d(dh), torch.zeros(N, OC // 2, dtype=torch.float64))
    assert torch.equal(d(dp), dp64)
    want, mag = dp64 @ mats, dp64.abs() @ mats.abs()
    within(dx, want, (sum_error(OC) + HALF + 2.0 ** -17) * mag + 2 * TINY * dp64.abs().sum(1, keepdim=True) + HALF * want.abs() + TINY)


def bank(seed, slots, R, OC, IC):
    a, b = randn(seed, slots, R, IC, scale=IC ** -0.5), randn(seed + 1, slots, OC, R, scale=0.5 * R ** -0.5)
    return a, b, torch.linspace(0.25, 2.0, slots, device=DEV)


def adapters64(w, x, bias, a, b, s, index):
    """Output and tolerance: the layer rounded to fp16, the rank sums to 2^-11 of the row's largest (they are held in fp16 with a common exponent: half a step of any of them is at most that), the sum
    rounded once more."""
    y, err = preacts(w, x, bias)
    delta, slack = torch.zeros_like(y), torch.zeros_like(y)
    x, a, b, s = d(x), d(a), d(b), d(s)
    for n, i in enumerate(index.tolist()):
        if 0 <= i < a.shape[0]:
            t, mag = a[i] @ x[n], a[i].abs() @ x[n].abs()
            et = sum_error(w.IC) * mag + HALF * t.abs().max()
            delta[n] = s[i] * (b[i] @ t)
            slack[n] = s[i].abs() * (b[i].abs() @ (et + sum_error(t.numel()) * t.abs()))
    out = y + delta
    base = err * (1 + HALF) + HALF * y.abs() + TINY
    return out, (base + slack + 2.0 ** -22 * (y.abs() + delta.abs())) * (1 + HALF) + HALF * out.abs() + TINY


ADAPTERS = [(3, 2, 256, 64, 1, 8, 1, False), (2, 2, 512, 320, 2, 16, 3, True), (2, 1, 256, 1024, 9, 24, 5, False), (2, 3, 768, 576, 16, 64, 40, True), (3, 2, 512, 512, 17, 40, 3, False),
            (3, 2, 1024, 256, 50, 128, 4, True), (2, 2, 512, 832, 130, 256, 2, False), (2, 1, 768, 448, 300, 32, 7, True), (2, 3, 256, 1344, 1200, 72, 3, False), (3, 2, 512, 256, 257, 8, 300, False),
            (2, 2, 256, 576, 700, 200, 90, True)]


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,R,slots,bias", ADAPTERS)
@pytest.mark.parametrize("order", ["mixed", "runs"])
def test_adapters(E, M, OC, IC, N, R, slots, bias, order):
    w = Weight(OC + IC + N, E, M, OC, IC, groups=bias)
    x, c = randn(N, N, IC), randn(N + 1, OC, scale=0.3) if bias else None
    a, b, s = bank(N + 2, slots, R, OC, IC)
    index = torch.randint(-1, slots, (N,), generator=torch.Generator().manual_seed(N), dtype=torch.int32)
    index = index.sort().values.flip(0) if order == "runs" else index
    want, tol = adapters64(w, x, c, a, b, s, index)
    for splitK in (None, 2):
        got = fp6.adapter_forward_native(E, M, x, w.native, w.scales, OC, a, b, s, index.to(DEV), splitK=splitK, group_exps=w.exps, bias=c)
        within(got, want, tol, "splitK %s" % splitK)


@gpu
def test_adapter_numbers_that_are_no_slots():
    """Rows without an adapter get the layer's own bits, whatever number says so and whatever the slots hold that nobody uses."""
    w = Weight(5, 3, 2, 512, 640)
    a, b, s = bank(6, 4, 16, 512, 640)
    a[1], b[1], s[1] = float("nan"), float("inf"), float("nan")
    for N in (1, 16, 21, 90):
        x = randn(N, N, 640)
        plain = fp6.linear_forward_native(3, 2, x, w.native, w.scales, 512)
        for number in (-1, -2 ** 31, 4, 2 ** 31 - 1):
            got = fp6.adapter_forward_native(3, 2, x, w.native, w.scales, 512, a, b, s, torch.full((N,), number, dtype=torch.int32, device=DEV), splitK=1)
            assert torch.equal(got, plain), (N, number)
        index = torch.arange(N, dtype=torch.int32) % 4
        index[index == 1] = -1
        want, tol = adapters64(w, x, None, a, b, s, index)
        within(fp6.adapter_forward_native(3, 2, x, w.native, w.scales, 512, a, b, s, index.to(DEV)), want, tol)


@gpu
def test_adapters_keep_requests_apart():
    """An adapter with infinities, and a row with a NaN, touch the rows that use them alone; a large and a tiny rank sum are both exact to their own size."""
    w = Weight(5, 2, 2, 256, 256)
    a, b, s = bank(6, 3, 8, 256, 256)
    x = randn(9, 18, 256)
    index = torch.tensor([0, 1, 2] * 6, dtype=torch.int32)
    clean = fp6.adapter_forward_native(2, 2, x, w.native, w.scales, 256, a, b, s, index.to(DEV))
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1, 3], b2[1, 200], x2[0, 5] = float("inf"), float("nan"), float("nan")
    got = fp6.adapter_forward_native(2, 2, x2, w.native, w.scales, 256, a2, b2, s, index.to(DEV))
    keep = [n for n in range(18) if index[n] != 1 and n != 0]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[0]).all()
    big, small = a.clone(), a.clone()
    big[0] *= 3000    # rank sums of some thousands times |x|: beyond fp16 with |x| = 60
    small[2] *= 2.0 ** -9
    for bk, xs, bs in ((big, 60.0, 1e-4), (small, 2.0 ** -6, 64.0)):
        xx, bb = (x.float() * xs).half(), (b.float() * bs).half()
        want, tol = adapters64(w, xx, None, bk, bb, s, index)
        got = fp6.adapter_forward_native(2, 2, xx, w.native, w.scales, 256, bk, bb, s, index.to(DEV))
        within(got, want, tol)


@gpu
@pytest.mark.parametrize("N,R", [(130, 40), (300, 16), (300, 72)])
def test_adapters_keep_requests_apart_in_large_tiles(N, R):
    """The same where a tile of 64 rows holds many adapters, and rows without one: those get the layer's own bits."""
    w = Weight(5, 2, 2, 512, 320)
    a, b, s = bank(6, 7, R, 512, 320)
    x, index = randn(9, N, 320), torch.randint(-1, 7, (N,), generator=torch.Generator().manual_seed(R), dtype=torch.int32)
    clean = fp6.adapter_forward_native(2, 2, x, w.native, w.scales, 512, a, b, s, index.to(DEV), splitK=1)
    assert torch.equal(clean[index < 0], fp6.linear_forward_native(2, 2, x, w.native, w.scales, 512)[index < 0])
    a2, b2, s2, x2 = a.clone(), b.clone(), s.clone(), x.clone()
    a2[1, 3], b2[2, 200, 5], s2[3] = float("inf"), float("nan"), float("inf")
    row = int((index == 4).nonzero()[0])
    x2[row, 5] = float("nan")
    buf = torch.full((N + 2, 512), 7.0, dtype=torch.float16, device=DEV)
    got = fp6.adapter_forward_native(2, 2, x2, w.native, w.scales, 512, a2, b2, s2, index.to(DEV), splitK=1, out=buf[:N])
    keep = [n for n in range(N) if index[n] not in (1, 2, 3) and n != row]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[row]).all() and (buf[N:] == 7.0).all()
    assert not torch.isfinite(got[index == 1]).any() and torch.isnan(got[index == 2][:, 200]).all() and not torch.isfinite(got[index == 3]).any()
    others = [c for c in range(512) if c != 200]
    assert torch.equal(got[index == 2][:, others], clean[index == 2][:, others])


@gpu
def test_strided_activations_given_outputs_and_another_stream():
    w = Weight(3, 3, 2, 512, 320, True)
    N = 70
    x, dy = randn(1, N, 640)[:, ::2], randn(2, 512, N).t()
    a, b, s = bank(3, 3, 16, 512, 320)
    index = (torch.arange(N, device=DEV) % 4 - 1).int()
    args = (3, 2, x.contiguous(), w.native, w.scales, 512)
    pre = torch.empty(N, 512, device=DEV)
    dh = dy[:, :256].contiguous()
    wants = [fp6.gated_forward_native(*args, preact=pre, group_exps=w.exps), fp6.linear_input_grad_native(3, 2, dy.contiguous(), w.native, w.scales, 320, group_exps=w.exps),
             fp6.adapter_forward_native(*args, a, b, s, index, group_exps=w.exps), *fp6.gated_backward_native(3, 2, dh, pre, w.native, w.scales, 320, group_exps=w.exps)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [torch.empty_like(t) for t in wants]
        args = (3, 2, x, w.native, w.scales, 512)
        got = [fp6.gated_forward_native(*args, group_exps=w.exps, out=outs[0]), fp6.linear_input_grad_native(3, 2, dy, w.native, w.scales, 320, group_exps=w.exps, out=outs[1]),
               fp6.adapter_forward_native(*args, a, b, s, index, group_exps=w.exps, out=outs[2]),
               *fp6.gated_backward_native(3, 2, dy[:, :256], pre, w.native, w.scales, 320, group_exps=w.exps, grad_in=outs[3], grad_preact=outs[4])]
    side.synchronize()
    for g, o, t in zip(got, outs, wants):
        assert g is o and torch.equal(g, t)


@gpu
@pytest.mark.parametrize("N", [4, 40, 150])
def test_captured_calls_replay_to_the_eager_results(N):
    """Two graphs of all operators on one stream, replayed in turn with eager calls of other sizes between them, on inputs that change."""
    OC, IC = 512, 1088
    w = Weight(3, 3, 2, OC, IC)
    a, b, s = bank(3, 3, 16, OC, IC)
    index = (torch.arange(N, device=DEV) % 4 - 1).int()

    def run(x, dh, splitK):
        pre = torch.empty(N, OC, device=DEV)
        h = fp6.gated_forward_native(3, 2, x, w.native, w.scales, OC, splitK=splitK, preact=pre)
        y = fp6.adapter_forward_native(3, 2, x, w.native, w.scales, OC, a, b, s, index, splitK=splitK)
        return (h, y, pre) + fp6.gated_backward_native(3, 2, dh, pre, w.native, w.scales, IC, splitK=splitK) + \
            (fp6.gated_forward_native(3, 2, x, w.native, w.scales, OC), fp6.linear_input_grad_native(3, 2, y, w.native, w.scales, IC))
    x, dh = randn(1, N, IC), randn(2, N, OC // 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        run(x, dh, 2)
        torch.cuda.synchronize()
        for splitK in (2, 4):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = run(x, dh, splitK)
            graphs.append((graph, outs, splitK))
        for seed in range(3):
            x.copy_(randn(10 + seed, N, IC))
            dh.copy_(randn(20 + seed, N, OC // 2))
            for graph, outs, splitK in graphs:
                want = [t.clone() for t in run(x, dh, splitK)]
                graph.replay()
                fp6.gated_forward_native(3, 2, randn(5, 300, IC), w.native, w.scales, OC, splitK=3)   # (eager work behind it, in the eager workspace)
                torch.cuda.synchronize()
                assert all(torch.equal(g, t) for g, t in zip(outs, want)), (seed, splitK)


@gpu
def test_calls_of_two_threads_on_one_stream():
    import threading
    w = Weight(3, 3, 2, 512, 1088)
    a, b, s = bank(3, 3, 16, 512, 1088)
    xs, idx = [randn(i, 20, 1088) for i in range(2)], (torch.arange(20, device=DEV) % 4 - 1).int()
    call = lambda x: fp6.adapter_forward_native(3, 2, x, w.native, w.scales, 512, a, b, s, idx, splitK=2)   # noqa: E731
    wants, results = [call(x) for x in xs], [[], []]
    threads = [threading.Thread(target=lambda i=i: [results[i].append(call(xs[i])) for _ in range(50)]) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for got, want in zip(results, wants):
        assert len(got) == 50 and all(torch.equal(g, want) for g in got)


def test_pair_order():
    g, u = torch.arange(48).reshape(48, 1).expand(48, 3), 100 + torch.arange(48).reshape(48, 1).expand(48, 3)
    p = fp6.gate_up_pairs(g, u)
    assert p.shape == (96, 3) and p[:, 0].tolist() == [*range(16), *range(100, 116), *range(16, 32), *range(116, 132), *range(32, 48), *range(132, 148)]
    with pytest.raises(ValueError):
        fp6.gate_up_pairs(g, u[:32])
    with pytest.raises(ValueError):
        fp6.gate_up_pairs(g[:8], u[:8])
    # native layouts: the same as the native layout of the rows in pair order
    rng = np.random.default_rng(0)
    codes = [rng.integers(0, 32, (64, 320)).astype(np.uint8) for _ in range(2)]
    nat = [fp6.weight_prepacking_native_cpu(2, 2, torch.from_numpy(quant.pack_raw(c, 2, 2))) for c in codes]
    both = fp6.gate_up_pairs(*(torch.from_numpy(c) for c in codes)).numpy()
    assert torch.equal(fp6.gate_up_pairs(*nat, rows=64), fp6.weight_prepacking_native_cpu(2, 2, torch.from_numpy(quant.pack_raw(both, 2, 2))))


def test_refusals_of_the_c_abi():
    """Status codes on arguments that no launch follows (the pointers are never read)."""
    L, p = _lib.lib(), 1 << 20
    grad = lambda E=3, M_=2, W=p, sc=p, ge=None, dy=p, dx=p, OC=256, N=4, IC=64, ws=None, s=1: L.fp6mi_linear_grad_native(E, M_, None, W, sc, ge, dy, dx, OC, N, IC, ws, s)   # noqa: E731
    assert grad(E=4) == -1 and grad(OC=128) == -2 and grad(IC=32) == -2 and grad(N=0) == -2 and grad(W=None) == -3 and grad(dx=None) == -3
    assert grad(s=2) == -4 and grad(s=0) == -5 and grad(dy=p + 8) == -6 and grad(ge=p + 1) == -6 and grad(OC=(1 << 20) + 256) == -2
    gated = lambda act=0, x=p, h=p, pre=None, ws=p, s=1, OC=256, bias=None: L.fp6mi_gated_native(3, 2, None, p, p, None, bias, x, h, pre, OC, 4, 64, act, ws, s)   # noqa: E731
    assert gated(act=3) == -9 and gated(act=-1) == -9 and gated(OC=0) == -2 and gated(x=None) == -3 and gated(h=None) == -3 and gated(pre=p + 2) == -6 and gated(bias=p + 1) == -6
    assert gated(s=2, ws=None) == -4 and gated(s=0) == -5 and L.fp6mi_query_gated_launch(3, 2, 256, 4, 64, 0, None) == -3
    back = lambda act=0, dh=p, pre=p, dp=p, dx=p, ws=p, s=1: L.fp6mi_gated_backward_native(3, 2, None, p, p, None, dh, pre, dp, dx, 256, 4, 64, act, ws, s)   # noqa: E731
    assert back(act=9) == -9 and back(dh=None) == -3 and back(pre=None) == -3 and back(ws=None) == -4 and back(dx=None) == -3 and back(dh=p + 4) == -6 and back(dp=p + 4) == -6 and back(s=0) == -5
    lora = lambda a=p, b=p, sc=p, ix=p, R=16, slots=2, ws=p, s=1: L.fp6mi_adapter_native(3, 2, None, p, p, None, None, p, p, a, b, sc, ix, 256, 4, 64, R, slots, ws, s)   # noqa: E731
    assert lora(a=None) == -3 and lora(b=None) == -3 and lora(sc=None) == -3 and lora(ix=None) == -3 and lora(ws=None) == -4 and lora(R=12) == -2 and lora(R=0) == -2 and lora(R=264) == -2
    assert lora(slots=0) == -2 and lora(a=p + 8) == -6 and lora(sc=p + 2) == -6 and lora(ix=p + 1) == -6
    assert b"activation" in L.fp6mi_error_string(-9)
    assert L.fp6mi_grad_workspace_bytes(10, 64, 1) == 0 and L.fp6mi_grad_workspace_bytes(10, 64, 3) == 3 * 10 * 64 * 4


def test_shapes_of_the_gated_block_beyond_the_wide_tiles():
    """The wide tiles take up to 2^20 columns; longer rows have another kernel for every batch, not a refusal."""
    import ctypes
    L, shape = _lib.lib(), (ctypes.c_int * 5)()
    for OC in (256, 768, 2048, 5120, 22016):
        for N in (1, 17, 40, 100, 145, 200, 300, 513, 1000, 4000):
            for IC in ((1 << 20) + 64, (1 << 21) + 192):
                for groups in (0, 1):
                    assert L.fp6mi_query_gated_launch(3, 2, OC, N, IC, groups, shape) == 0
                    kind, nt, rt, wr, wk = shape
                    assert kind < 2 or wk == 4, (OC, N, IC, list(shape))


def test_grad_splits_are_in_range():
    L = _lib.lib()
    for OC in (256, 4096, 28672):
        for IC in (64, 1024, 8192):
            for N in (1, 16, 100, 5000):
                assert 1 <= L.fp6mi_heuristic_grad_splits(3, 2, OC, N, IC, 256) <= max(1, OC // 32)
    assert L.fp6mi_heuristic_grad_splits(3, 2, 0, 1, 64, 256) == 1
    rows = [L.fp6mi_query_grad_launch(E, M, OC, N, IC, s) for E, M, OC, IC, N, _ in GRAD for s in (1, 3)]
    assert set(rows) == {16, 32, 128, 192, 256}   # the cases above reach every kernel
    assert L.fp6mi_query_grad_launch(4, 4, 256, 1, 64, 1) == -1 and L.fp6mi_query_grad_launch(3, 2, 128, 1, 64, 1) == -2 and L.fp6mi_query_grad_launch(3, 2, 256, 1, 64, 0) == -5


@gpu
def test_refusals_of_the_python_functions():
    w = Weight(3, 3, 2, 512, 320)
    x, a, b, s = randn(1, 6, 320), randn(2, 3, 16, 320), randn(3, 3, 512, 16), torch.ones(3, device=DEV)
    idx = torch.zeros(6, dtype=torch.int32, device=DEV)
    gated = lambda x=x, OC=512, **kw: fp6.gated_forward_native(3, 2, x, w.native, w.scales, OC, **kw)   # noqa: E731
    for kw in (dict(x=x.float()), dict(x=x.cpu()), dict(x=x[0]), dict(x=x[:0]), dict(OC=256), dict(OC=500), dict(activation="relu"), dict(activation=None), dict(splitK=0),
               dict(out=torch.empty(6, 512, dtype=torch.float16, device=DEV)), dict(preact=torch.empty(6, 256, device=DEV)),
               dict(preact=torch.empty(6, 512, dtype=torch.float16, device=DEV)), dict(bias=torch.empty(256, dtype=torch.float16, device=DEV)), dict(group_exps=torch.empty(4, dtype=torch.uint8, device=DEV)),
               dict(splitK=2, workspace=torch.empty(10, device=DEV)), dict(x=randn(1, 6, 256))):
        with pytest.raises(ValueError):
            gated(**kw)
    lora = lambda a=a, b=b, s=s, idx=idx, **kw: fp6.adapter_forward_native(3, 2, x, w.native, w.scales, 512, a, b, s, idx, **kw)   # noqa: E731
    for kw in (dict(a=a.float()), dict(a=a[:2]), dict(a=a[:, :12]), dict(a=a[0]), dict(a=a.cpu()), dict(b=b[:, :256]), dict(b=b.transpose(1, 2)), dict(s=s[:2]), dict(s=s.half()),
               dict(idx=idx.long()), dict(idx=idx[:5]), dict(idx=idx.cpu()), dict(idx=idx.repeat(2)[::2]), dict(a=a[:0], b=b[:0], s=s[:0]), dict(workspace=torch.empty(1, device=DEV))):
        with pytest.raises(ValueError):
            lora(**kw)
    dy, pre, dh = randn(4, 6, 512), randn(5, 6, 512).float(), randn(6, 6, 256)
    for kw in (dict(grad_out=dy.float()), dict(grad_out=dy[:, :256]), dict(IC=256), dict(IC=300), dict(splitK=-1), dict(out=torch.empty(6, 256, dtype=torch.float16, device=DEV))):
        with pytest.raises(ValueError):
            fp6.linear_input_grad_native(3, 2, **{**dict(grad_out=dy, native_weight=w.native, scales=w.scales, IC=320), **kw})
    for kw in (dict(grad_out=dh[:5]), dict(grad_out=dy), dict(preact=pre[:, :256]), dict(preact=pre.half()), dict(activation="tanh"), dict(grad_preact=dh), dict(grad_in=dh)):
        with pytest.raises(ValueError):
            fp6.gated_backward_native(3, 2, **{**dict(grad_out=dh, preact=pre, native_weight=w.native, scales=w.scales, IC=320), **kw})
    with pytest.raises(ValueError):
        fp6.linear_input_grad_native(5, 2, dy, w.native, w.scales, 320)
    with pytest.raises(fp6.Fp6miError):   # a view that starts between two 16-byte boundaries
        gated(x=randn(1, 6 * 320 + 4)[4:].view(6, 320))


# ---- every launch shape ----
GATED_SHAPES = [  # one problem for every launch shape of the gated block, with and without group exponents: E, M, OC, IC, N, activation, group exponents, bias
    (3, 2, 256, 576, 1, "silu", False, True), (2, 2, 256, 576, 1, "gelu", True, True), (2, 3, 256, 1088, 1, "gelu_tanh", False, False),
    (2, 1, 256, 1088, 1, "silu", True, False), (3, 2, 256, 2112, 1, "gelu", False, True), (2, 2, 256, 2112, 1, "gelu_tanh", True, True),
    (2, 3, 8448, 576, 5, "silu", False, False), (2, 1, 8448, 576, 5, "gelu", True, False), (3, 2, 256, 1088, 513, "gelu_tanh", False, True),
    (2, 2, 256, 1088, 513, "silu", True, True), (2, 3, 16640, 576, 5, "gelu", False, False), (2, 1, 16640, 576, 5, "gelu_tanh", True, False),
    (3, 2, 4352, 1408, 49, "silu", False, True), (2, 2, 4352, 1408, 49, "gelu", True, True), (2, 3, 24832, 576, 5, "gelu_tanh", False, False),
    (2, 1, 24832, 576, 5, "silu", True, False), (3, 2, 6400, 5312, 17, "gelu", False, True), (2, 3, 6400, 5312, 17, "gelu_tanh", True, True),
    (3, 2, 12544, 1408, 25, "silu", False, False), (2, 3, 12544, 1408, 25, "gelu", True, False), (2, 2, 5632, 1408, 33, "gelu_tanh", False, True),
    (3, 2, 5632, 1408, 33, "silu", True, True), (2, 1, 17408, 1728, 17, "gelu", False, False), (2, 2, 17408, 1728, 17, "gelu_tanh", True, False),
    (2, 3, 13312, 6272, 33, "silu", False, True), (3, 2, 13312, 6272, 33, "gelu", True, True), (2, 1, 768, 576, 1345, "gelu_tanh", False, False),
    (2, 2, 768, 576, 1345, "silu", True, False), (2, 1, 256, 576, 2049, "gelu", False, True), (2, 2, 256, 576, 2049, "gelu_tanh", True, True),
    (2, 3, 256, 832, 17, "silu", False, False), (2, 1, 256, 832, 17, "gelu", True, False), (2, 1, 15360, 2752, 81, "gelu_tanh", False, True),
    (3, 2, 33280, 2112, 33, "silu", True, True), (2, 3, 8192, 1408, 193, "gelu", False, False), (3, 2, 8192, 1408, 193, "gelu_tanh", True, False),
    (2, 2, 22016, 576, 65, "silu", False, True), (2, 3, 22016, 576, 65, "gelu", True, True), (2, 2, 22016, 1408, 129, "gelu_tanh", False, False),
    (2, 1, 22016, 1408, 129, "silu", True, False), (3, 2, 22016, 1408, 161, "gelu", False, True), (2, 2, 22016, 1408, 161, "gelu_tanh", True, True),
    (2, 1, 768, 1728, 513, "silu", False, False), (2, 2, 1280, 1408, 385, "gelu", True, False), (2, 3, 5632, 1408, 65, "gelu_tanh", False, True),
    (3, 2, 5632, 1408, 65, "silu", True, True), (2, 3, 1280, 1408, 385, "gelu", False, False), (2, 1, 1280, 1408, 385, "gelu_tanh", True, False),
    (3, 2, 2304, 1408, 321, "silu", False, True), (2, 2, 2304, 1408, 321, "gelu", True, True), (2, 3, 5632, 1408, 321, "gelu_tanh", False, False),
    (2, 2, 4864, 1408, 391, "silu", True, False), (3, 2, 768, 1088, 2689, "gelu", False, True), (2, 3, 8448, 1088, 193, "gelu_tanh", True, True),
    (2, 1, 16640, 1408, 65, "silu", False, False), (3, 2, 6144, 1408, 257, "gelu", True, False), (2, 1, 22016, 1088, 129, "gelu_tanh", False, True),
    (2, 2, 22016, 1088, 129, "silu", True, True), (2, 3, 11008, 576, 129, "gelu", False, False), (2, 1, 11008, 576, 129, "gelu_tanh", True, False),
    (3, 2, 16640, 1408, 81, "silu", False, True), (2, 2, 16640, 1408, 81, "gelu", True, True), (2, 3, 22016, 576, 129, "gelu_tanh", False, False),
    (2, 1, 22016, 576, 129, "silu", True, False), (2, 2, 1792, 1088, 2881, "gelu", False, True), (2, 1, 1792, 1088, 2881, "gelu_tanh", True, True),
    (3, 2, 8192, 1088, 385, "silu", False, False), (2, 3, 8192, 1088, 385, "gelu", True, False), (2, 1, 33024, 1344, 97, "gelu_tanh", False, True),
    (3, 2, 7424, 1088, 769, "silu", True, True), (2, 2, 16640, 576, 97, "gelu", False, False), (2, 3, 16640, 576, 97, "gelu_tanh", True, False),
    (3, 2, 43776, 576, 65, "silu", False, True), (2, 2, 43776, 576, 65, "gelu", True, True), (2, 3, 33024, 576, 97, "gelu_tanh", False, False),
    (3, 2, 33024, 576, 97, "silu", True, False)]


def gated_shape(E, M, OC, IC, N, groups):
    import ctypes
    shape = (ctypes.c_int * 5)()
    assert _lib.lib().fp6mi_query_gated_launch(E, M, OC, N, IC, int(groups), shape) == 0
    return tuple(shape)


def test_gated_shapes_are_all_there_are():
    """The problems above reach every launch shape that sizes from the smallest to the largest ask for, and the kernels are compiled for no other."""
    reached = {(gated_shape(E, M, OC, IC, N, groups), groups) for E, M, OC, IC, N, _, groups, _ in GATED_SHAPES}
    asked = set()
    for E, M in FORMATS:
        for OC in (256, 768, 1280, 2304, 4096, 5632, 6400, 8192, 12544, 13312, 16640, 17408, 22016, 28672, 33024, 43776, 57344):
            for IC in (64, 576, 1088, 1408, 1536, 2752, 4096, 5312, 6272, 8192, 11008, 28672):
                for N in (1, 2, 5, 8, 9, 16, 17, 24, 25, 32, 33, 40, 49, 64, 65, 72, 81, 96, 97, 112, 129, 145, 161, 193, 225, 257, 321, 385, 513, 769, 1024, 1345, 2048, 2049, 2689, 2881, 4096):
                    asked |= {(gated_shape(E, M, OC, IC, N, groups), groups) for groups in (False, True)}
    assert reached == asked and len(GATED_SHAPES) == len(reached)
    import os
    import re
    with open(os.path.join(os.path.dirname(fp6.__file__), "csrc", "fp6mi_block.hip")) as f:
        text = f.read()
    instances = text[text.index("int gated_cfg("):text.index("int op_gated(")]
    assert len(re.findall(r"FP6MI_CASE\(\d", instances)) == len({shape for shape, _ in reached})


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,act,groups,bias", GATED_SHAPES, ids=lambda v: str(v))
def test_gated_block_in_every_shape(E, M, OC, IC, N, act, groups, bias):
    w = Weight(OC + IC + N, E, M, OC, IC, groups)
    x, b = randn(N, N, IC), randn(N + 1, OC, scale=0.3) if bias else None
    y, err, h, tol = gated64(w, x, b, act)
    buf, pre = torch.full((N + 2, OC // 2), 7.0, dtype=torch.float16, device=DEV), torch.full((N + 2, OC), 7.0, device=DEV)
    fp6.gated_forward_native(E, M, x, w.native, w.scales, OC, act, out=buf[:N], preact=pre[:N], group_exps=w.exps, bias=b)
    within(buf[:N], h, tol, "out")
    within(pre[:N], y, err, "preact")
    assert (buf[N:] == 7.0).all() and (pre[N:] == 7.0).all()
    assert torch.equal(fp6.gated_forward_native(E, M, x, w.native, w.scales, OC, act, group_exps=w.exps, bias=b), buf[:N])


BACKWARD = [  # E, M, OC, IC, N, splits, group exponents: every kernel of the input gradient behind gated_grad, which hands it products with the mantissas
    (3, 2, 512, 320, 9, 1, True), (2, 1, 1024, 448, 13, 3, False), (2, 2, 512, 576, 27, 2, False), (2, 3, 768, 320, 31, 1, True), (2, 2, 1024, 320, 130, 1, False), (3, 2, 512, 704, 99, 3, True),
    (3, 2, 256, 4928, 1537, 1, True), (2, 1, 512, 7232, 258, 3, False), (2, 3, 512, 6528, 130, 5, True), (2, 2, 256, 6528, 521, 2, False),
    (2, 2, 512, 7232, 1558, 1, True), (2, 3, 512, 7296, 391, 3, False), (3, 2, 512, 6464, 194, 5, False), (2, 1, 256, 6464, 791, 2, True)]


def test_gradient_kernels_behind_the_block():
    rows = {(_lib.lib().fp6mi_query_grad_launch(E, M, OC, N, IC, s), s > 1, groups) for E, M, OC, IC, N, s, groups in BACKWARD}
    assert {r for r, _, _ in rows} == {16, 32, 128, 192, 256}
    assert {r[:2] for r in rows} == {(r, s) for r in (16, 32, 128, 192, 256) for s in (False, True)}
    assert {r[::2] for r in rows} == {(r, g) for r in (16, 32, 128, 192, 256) for g in (False, True)}


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,splits,groups", BACKWARD)
def test_gated_block_backward_by_every_kernel(E, M, OC, IC, N, splits, groups):
    w = Weight(OC + IC + N, E, M, OC, IC, groups)
    dh, pre = randn(3, N, OC // 2, scale=0.1), randn(4, N, OC).float()
    buf = torch.full((N + 2, IC), 7.0, dtype=torch.float16, device=DEV)
    dx, dp = fp6.gated_backward_native(E, M, dh, pre, w.native, w.scales, IC, "gelu", splitK=splits, grad_in=buf[:N], group_exps=w.exps)
    (g, u), dd = halves(d(pre)), d(dh)
    want = pairs(dd * u * slope64("gelu", g), dd * act64("gelu", g))
    slack = 2.0 ** -18 * pairs(dd.abs() * u.abs() * (1 + g.abs()), dd.abs() * g.abs())   # (slopes and activations as in the test above)
    within(dp, want, HALF * want.abs() + slack + TINY, "grad_preact")
    # a product of dp with a mantissa (1/2 and up: below the normal halfs half a step is 2 * TINY of the weight) is rounded once; its float32 value is off by the slack and two roundings more
    dx64, mag = want @ w.w, want.abs() @ w.w.abs()
    within(dx, dx64, (sum_error(OC + 2) + HALF) * mag + (slack + 2 * TINY) @ w.w.abs() * (1 + HALF) + HALF * dx64.abs() + TINY, "grad_in")
    assert (buf[N:] == 7.0).all()


@gpu
@pytest.mark.parametrize("N,R", [(1, 8), (1, 72), (16, 16), (47, 40), (112, 72), (256, 32)])
def test_rank_sums_of_few_rows_are_held_as_two_halfs(N, R):
    """Beside a layer of zeros the output is the adapter's part alone, rounded once; of a row with one value a rank sum is one product, exact in float32, and so are its halfs' products with b.  Tiles
    of sixteen rows hold it to 2^-22 of itself (two halfs), or 2^-39 of the row's largest (half a step below the normal halfs, where that one is from 2^14 to 2^15).  One half would be off by more than
    that allows."""
    OC, IC, slots = 256, 64, 3
    w = Weight(5, 3, 2, OC, IC)
    a, b, s = bank(6, slots, R, OC, IC)
    x, index = torch.zeros(N, IC, dtype=torch.float16, device=DEV), torch.arange(N, dtype=torch.int32) % slots
    x[torch.arange(N), torch.arange(N) * 7 % IC] = randn(N, N)
    got = fp6.adapter_forward_native(3, 2, x, w.native, torch.zeros_like(w.scales), OC, a, b, s, index.to(DEV))
    i = index.long()
    t = torch.stack([d(a)[i[n]] @ d(x)[n] for n in range(N)])
    top = t.abs().amax(1, keepdim=True)
    et = 2.0 ** -22 * t.abs() + 2.0 ** -39 * top
    part = lambda m, v: torch.stack([m[i[n]] @ v[n] for n in range(N)]) * d(s)[i][:, None]   # noqa: E731
    want = part(d(b), t)
    slack = part(d(b).abs(), et + sum_error(2 * R + 2) * t.abs())
    within(got, want, slack * (1 + HALF) + HALF * want.abs() + TINY)
    power = torch.exp2(torch.floor(torch.log2(top)) - 14)
    one = part(d(b), (t / power).half().double() * power)   # (what one half a sum would give: the bound tells them apart)
    assert ((one - want).abs() > 2 * slack).any()


@gpu
@pytest.mark.parametrize("N", [3, 50, 300])
def test_calls_without_the_extension(N, monkeypatch):
    """ctypes and the extension launch the same kernels with the same splits, and refuse the same calls."""
    assert fp6._ext is not None
    w = Weight(3, 2, 2, 512, 1344, True)
    x, dy, dh, c = randn(1, N, 1344), randn(2, N, 512), randn(3, N, 256), randn(4, 512)
    a, b, s = bank(3, 3, 16, 512, 1344)
    index = (torch.arange(N, device=DEV) % 4 - 1).int()
    fmt, got = (2, 2), []
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        for split in (None, 2):
            pre = torch.empty(N, 512, device=DEV)
            got.append([fp6.gated_forward_native(*fmt, x, w.native, w.scales, 512, "gelu", splitK=split, preact=pre, group_exps=w.exps, bias=c), pre,
                        *fp6.gated_backward_native(*fmt, dh, pre, w.native, w.scales, 1344, "gelu", splitK=split, group_exps=w.exps),
                        fp6.linear_input_grad_native(*fmt, dy, w.native, w.scales, 1344, splitK=split, group_exps=w.exps),
                        fp6.adapter_forward_native(*fmt, x, w.native, w.scales, 512, a, b, s, index, splitK=split, group_exps=w.exps, bias=c)])
        assert fp6.gated_backward_native(*fmt, dh, pre, w.native, w.scales, 1344, grad_preact=False, group_exps=w.exps)[1] is None
    for ours, theirs in zip(got[:2], got[2:]):
        assert all(torch.equal(p, q) for p, q in zip(ours, theirs))
    if N == 3:   # (without the extension from here on)
        test_refusals_of_the_python_functions()


@gpu
def test_large_scratch_is_given_back(monkeypatch):
    """What a call keeps for the next one on its stream is bounded; partial sums and products beyond that are the call's own."""
    assert fp6._ext is not None
    OC, IC, N = 512, 8192, 2000
    w = Weight(1, 3, 2, OC, IC)
    dy, dh, pre, x = randn(1, N, OC), randn(2, N, OC // 2), randn(3, N, OC).float(), randn(4, N, IC)
    calls = [lambda: fp6.linear_input_grad_native(3, 2, dy, w.native, w.scales, IC, splitK=3), lambda: fp6.gated_backward_native(3, 2, dh, pre, w.native, w.scales, IC, splitK=3)[0],
             lambda: fp6.gated_forward_native(3, 2, x, w.native, w.scales, OC, splitK=30)]
    wants = [call().clone() for call in calls]
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        fp6.clear_caches()
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        for _ in range(2):
            for call, want in zip(calls, wants):
                assert torch.equal(call(), want)
        assert torch.cuda.memory_allocated() - held <= fp6.SPLIT_WORKSPACE_BYTES


# the projection down of a block: many columns, and so many ranges of them
@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,R,slots,bias", [(3, 2, 256, 28672, 1, 16, 3, False), (2, 2, 512, 11008, 20, 72, 5, True), (2, 1, 256, 11072, 33, 136, 4, False), (2, 3, 512, 28672, 120, 64, 30, True),
                                                      (3, 2, 256, 11008, 300, 24, 9, False), (2, 2, 512, 9152, 700, 40, 5, True)])
def test_adapters_of_long_rows(E, M, OC, IC, N, R, slots, bias):
    test_adapters(E, M, OC, IC, N, R, slots, bias, "mixed")


@gpu
@pytest.mark.parametrize("E,M,OC,IC,N,groups", [(3, 2, 512, 28672, 3, False), (2, 2, 1024, 11008, 29, True), (2, 3, 512, 11072, 100, False), (2, 1, 512, 28672, 333, True)])
def test_input_gradient_of_long_rows(E, M, OC, IC, N, groups):
    test_input_gradient(E, M, OC, IC, N, groups)
