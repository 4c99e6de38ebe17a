"""Products with 4-bit integer weights at the ends of their ranges: values, sizes, and calls that they have no part in."""
import pytest
import torch

import fp6_llm_amd as fp6
from test_int4 import DEV, KERNELS, TILES, Weight, by_kernel, choice, d, gated64, gpu, halves, randn, within

STREAMS = [k for k in range(len(KERNELS)) if k not in TILES]


def whole_numbers(w, seed, N, unit=1.0, device=DEV):
    """Rows of -1, 0 and 1 for a weight whose scales become 1 and 2 (times a power of two): sums of whole numbers, which float32 holds in any order as long as their magnitudes come to less than 2^24."""
    s = unit * torch.exp2(torch.randint(0, 2, w.scales.shape, generator=torch.Generator().manual_seed(seed)).double())
    each = torch.arange(w.IC) // w.group
    old = w.scales.cpu().double()
    w.w = (w.w / old[..., each]).round() * s[..., each]
    w.scales = s.to(w.dtype).to(device)
    w.native, w.native_scales = fp6.int4_pack_native(w.codes, w.scales, w.zeros, w.group)
    x = torch.randint(-1, 2, (N, w.IC), generator=torch.Generator().manual_seed(seed + 1)).double()
    assert w.E or float((x.abs() @ w.w.abs().t()).max()) < unit * 2 ** 24
    return x, w


# ---------------------------------------------------------------------------------------------------------------- whole numbers: every sum is exact, and an output off by anything is seen
EXACT = [  # OC, IC, N, group, zeros, type, the kernels that may be the choice
    (256, 8192, 1, 64, True, "bf16", STREAMS), (512, 4576, 16, 32, False, "bf16", STREAMS), (256, 28672, 2, 64, False, "fp16", STREAMS), (256, 28672, 70, 128, False, "bf16", range(12)), (4096, 4096, 16, 128, True, "fp16", STREAMS),
    (2064, 544, 31, 32, True, "bf16", STREAMS), (10240, 4576, 19, 32, True, "fp16", TILES), (4112, 11040, 64, 64, True, "fp16", TILES), (528, 1120, 65, 128, True, "bf16", STREAMS), (8208, 2080, 130, 128, False, "fp16", TILES),
    (4096, 4096, 256, 128, True, "bf16", TILES), (4112, 4128, 300, 32, True, "bf16", TILES), (8208, 2048, 777, 64, False, "bf16", TILES), (1072, 992, 513, 128, True, "fp16", STREAMS), (4112, 416, 1030, 64, False, "fp16", TILES), (2064, 28672, 150, 96, True, "bf16", TILES),
    (32, (1 << 20) + 160, 3, 128, True, "fp16", STREAMS), (32, (1 << 20) + 160, 40, 64, True, "bf16", STREAMS), (48, 1 << 19, 50, 128, False, "fp16", range(12))]


def native_group(group):
    return 128 if group % 128 == 0 else 64 if group % 64 == 0 else 32


@pytest.mark.parametrize("OC,IC,N,group,zeros,type,kernels", EXACT)
def test_whole_numbers_show_what_is_missing(OC, IC, N, group, zeros, type, kernels):
    """Of what is compared below: outputs of zeros, or without the last block of 128 columns (or what there is of it), the first group or one in the middle, are seen in most places; and the choice is what the case is there for."""
    x, w = whole_numbers(Weight(OC + IC + N, OC, IC, group, zeros, type, device="cpu"), OC, min(N, 16), device="cpu")
    assert choice(OC, N, IC, type, group=native_group(group)) in kernels
    want = x @ w.w.t()
    last = (IC - 1) // 128 * 128
    for columns in (slice(0, IC), slice(last, IC), slice(0, group), slice(IC // 2 // group * group, (IC // 2 // group + 1) * group)):
        part = x[:, columns] @ w.w[:, columns].t()
        assert (part != 0).double().mean() > 0.9, columns
        assert ((want - part).to(w.dtype) != want.to(w.dtype)).double().mean() > 0.6, columns   # (rounded outputs too)


@gpu
@pytest.mark.parametrize("OC,IC,N,group,zeros,type,kernels", EXACT)
def test_product_of_whole_numbers(OC, IC, N, group, zeros, type, kernels):
    x, w = whole_numbers(Weight(OC + IC + N, OC, IC, group, zeros, type), OC, N)
    want, x = x @ w.w.t(), x.to(w.dtype).to(DEV)
    b = torch.arange(OC).remainder(17).double() - 8
    assert torch.equal(fp6.int4_forward_native(x, w.native, w.native_scales).cpu(), want.to(w.dtype))
    got = fp6.int4_forward_native(x, w.native, w.native_scales, bias=b.to(w.dtype).to(DEV), out_dtype=torch.float32)
    assert torch.equal(d(got), want + b)


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("OC,IC,N,group,zeros,type,kernels", [(288, 28672, 7, 64, True, "bf16", STREAMS), (2080, 8192, 20, 32, False, "fp16", range(12)), (4096, 4096, 256, 128, True, "bf16", TILES), (4128, 8192, 70, 128, True, "fp16", TILES),
                                                              (544, 2080, 150, 32, True, "bf16", range(12))])
def test_gated_product_of_whole_numbers(act, OC, IC, N, group, zeros, type, kernels):
    """Exact pre-activations: what is left is the activation's own error (2^-18 of its argument) and the rounding."""
    assert choice(OC, N, IC, type, gated=True, group=native_group(group)) in kernels
    x, w = whole_numbers(Weight(OC + IC + N, OC, IC, group, zeros, type), OC, N, 2.0 ** -8)
    y, x = x @ w.w.t(), x.to(w.dtype).to(DEV)
    for dtype in (w.dtype, torch.float32):
        got = fp6.int4_forward_native(x, w.native, w.native_scales, activation=act, out_dtype=dtype)
        h, tol = gated64(y, torch.zeros_like(y), act, dtype)
        within(got, h, tol, str(dtype))
        g, u = halves(y)
        assert (h.abs() > 4 * tol)[(g > 0.5) & (u != 0)].all()   # (an output of zeros, or without the part of a column that is 2^-8 or more of it, is off by more)


@gpu
@pytest.mark.parametrize("T,k,E,OC,IC,group,zeros,type", [(1, 2, 8, 288, 11008, 128, False, "fp16"), (40, 8, 64, 288, 2080, 64, True, "bf16"), (700, 2, 8, 1056, 4128, 32, True, "fp16"), (1500, 2, 4, 2064, 2048, 128, True, "bf16"),
                                                          (320, 1, 64, 2048, 2560, 128, True, "fp16"), (320, 1, 64, 2048, 2560, 64, False, "bf16")])
def test_product_of_sorted_rows_of_whole_numbers(T, k, E, OC, IC, group, zeros, type):
    """Float32 outputs, as the product down of Int4Experts has them; the last two cases with all rows on one expert of many."""
    x, w = whole_numbers(Weight(T + OC + IC, OC, IC, group, zeros, type, E), E, T)
    assert 30 * IC < 2 ** 24
    g = torch.Generator().manual_seed(T)
    index = torch.full((T, k), 5) if T == 320 else torch.randint(-1, E, (T, k), generator=g)
    rows, plan = fp6.expert_sort(x.to(w.dtype).to(DEV), index.to(DEV), E)
    got = fp6.int4_forward_native(rows, w.native, w.native_scales, plan, out_dtype=torch.float32)
    rounded = fp6.int4_forward_native(rows, w.native, w.native_scales, plan)
    offsets, rows = plan.offsets.tolist(), d(rows)
    for e in range(E):
        want = rows[offsets[e]:offsets[e + 1]] @ w.w[e].t()
        assert torch.equal(d(got[offsets[e]:offsets[e + 1]]), want) and torch.equal(rounded[offsets[e]:offsets[e + 1]].cpu(), want.to(w.dtype)), e
    assert (got[offsets[-1]:] == 0).all() and (rounded[offsets[-1]:] == 0).all()


@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (96, True), (128, True), (128, False)])
@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_every_kernel_in_whole_numbers(kernel, type, group, zeros):
    if kernel == 10 and group != 128:
        pytest.skip("this kernel has groups of 128 only")
    cols = KERNELS[kernel][1]
    for OC, IC, N in ((48, 32, 1), (272, 96, cols), (96, 1184, cols + 1), (1056, 608, 2 * cols - 1), (32, 28704, 3), (288, 2048, 3 * cols + 5)):
        x, w = whole_numbers(Weight(OC + N + kernel, OC, IC, group, zeros, type), N, N)
        want, x = x @ w.w.t(), x.to(w.dtype).to(DEV)
        assert torch.equal(d(by_kernel(kernel, w, x, f32=True)), want) and torch.equal(by_kernel(kernel, w, x).cpu(), want.to(w.dtype)), (OC, IC, N)


# ---------------------------------------------------------------------------------------------------------------- infinities and large values
@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("kernel", STREAMS)
def test_bf16_rows_of_every_size_in_the_stream_kernels(kernel, group, zeros):
    """These multiply 16 + q, which leaves float32's range before q - z does: all that float32 sums of the weights' own products can hold comes out, and infinities as the definition has them.  Rows of
    whole numbers times a power of two, so that every sum is exact; of the last size 15 * 3 * 128 of a group's magnitudes come to 2^138."""
    w = Weight(5 + kernel, 80, 1184, group, zeros, "bf16")
    x, w = whole_numbers(w, 3, 9)
    w.native_scales = w.native_scales.clone()
    w.native_scales[..., 0] *= 2.0 ** -20   # (the numbers themselves are up to 2 * 15 * 1184, 2^-4 with these: all sums of scaled groups stay below 2^124)
    size = torch.tensor([0, 100, 120, 127, 127, 126, -100, 0, 0])
    x[:9] *= torch.exp2(size.double()).unsqueeze(1)
    want = x @ w.w.t() * 2.0 ** -20
    x[7, 5], x[8, 3], x[8, 40], x[4, 9] = float("inf"), float("inf"), float("-inf"), float("nan")
    got = d(by_kernel(kernel, w, x.bfloat16().to(DEV), f32=True))
    fine = [0, 1, 2, 3, 5, 6]
    assert torch.equal(got[fine], want[fine])
    assert got[4].isnan().all()
    # one infinity: of the weight's sign, a weight of zero makes NaN of it; two of opposite signs likewise where the weights have the same sign
    a, b, c = w.w[:, 5], w.w[:, 3], w.w[:, 40]
    assert torch.equal(got[7].isnan(), a == 0) and torch.equal(got[7][a != 0], a[a != 0].sign() * float("inf"))
    nan = (b == 0) | (c == 0) | (b.sign() == c.sign())
    assert torch.equal(got[8].isnan(), nan) and torch.equal(got[8][~nan], b[~nan].sign() * float("inf"))


@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("kernel", STREAMS)
def test_a_large_value_among_small_ones_costs_bf16_sums_nothing(kernel, group, zeros):
    """16 + q and 16 + z stand for q and z there: a group's sum is exact while 31 times its magnitudes come to less than 2^24, here 2^18 and up to 128 ones."""
    w = Weight(11 + kernel, 80, 1184, group, zeros, "bf16")
    x, w = whole_numbers(w, 5, 16)
    x[:, 70], x[:, 333] = 2.0 ** 18, -2.0 ** 17   # (in two groups; with scales of 1 and 2 all sums come to 2 * 15 * (2^18 + 2^17 + 1184) < 2^24 at the most)
    want = x @ w.w.t()
    assert torch.equal(d(by_kernel(kernel, w, x.bfloat16().to(DEV), f32=True)), want)


@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
@pytest.mark.parametrize("kernel", [k for k in range(len(KERNELS)) if k != 10])
def test_fp16_rows_of_every_size(kernel, group, zeros):
    """From the smallest number below the normal ones to the largest power of two; infinities and NaN as the definition has them."""
    w = Weight(7 + kernel, 96, 1184, group, zeros, "fp16")
    x, w = whole_numbers(w, 4, 9)
    x *= torch.exp2(torch.tensor([0, -24, -20, -15, -14, 15, 10, 0, 0]).double()).unsqueeze(1)
    want = x @ w.w.t()
    x[7, 5], x[8, 3], x[6, 1183] = float("inf"), float("nan"), 65504.0
    want[6] = x[6] @ w.w.t()
    assert float((x[6].abs() @ w.w.abs().t()).max()) < 2 ** 30   # (of multiples of 2^5: 2^24 of them, and 65504 is one)
    got = d(by_kernel(kernel, w, x.half().to(DEV), f32=True))
    assert torch.equal(got[:7], want[:7]) and got[8].isnan().all()
    a = w.w[:, 5]
    assert torch.equal(got[7].isnan(), a == 0) and torch.equal(got[7][a != 0], a[a != 0].sign() * float("inf"))


@gpu
@pytest.mark.parametrize("act", [None, "silu"])
def test_an_infinity_in_a_bf16_row_does_not_depend_on_how_many_rows_there_are(act):
    w = Weight(6, 4096, 512, 128, True, "bf16")
    x = randn(1, 2048, 512, dtype=torch.bfloat16)
    x[0, 7], x[0, 300] = float("inf"), 2.0 ** 122
    assert choice(4096, 1, 512, "bf16", gated=act is not None) in STREAMS and choice(4096, 2048, 512, "bf16", gated=act is not None) in TILES
    few, many = (fp6.int4_forward_native(x[:n], w.native, w.native_scales, activation=act, out_dtype=torch.float32)[0] for n in (1, 2048))
    assert torch.equal(few.isnan(), many.isnan()) and torch.equal(few[~few.isnan()], many[~many.isnan()]) and few.isinf().any()


# ---------------------------------------------------------------------------------------------------------------- what the product has no part in
def no_part_in(dev, monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx
    w = Weight(1, 32, 160, 32, True, device=dev)
    x, b = randn(1, 2, 160, device=dev), randn(2, 32, device=dev)
    call = lambda t: fp6.int4_forward_native(t, w.native, w.native_scales)   # noqa: E731
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        for bad in (dict(in_feats=x.clone().requires_grad_()), dict(bias=b.clone().requires_grad_()), dict(native_scales=w.native_scales.clone().requires_grad_())):
            with pytest.raises(ValueError, match="no gradient"):
                fp6.int4_forward_native(**{**dict(in_feats=x, native_weight=w.native, native_scales=w.native_scales, bias=b), **bad})
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
        for transform in (lambda: torch.func.vmap(call)(x.unsqueeze(0)), lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.vmap(lambda v: fp6.int4_forward_native(x, w.native, w.native_scales, bias=v))(b.unsqueeze(0))):
            with pytest.raises(RuntimeError, match="transform"):
                transform()
        with pytest.raises((RuntimeError, ValueError), match="transform|no gradient"):
            torch.func.grad(lambda t: call(t).float().sum())(x)
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (x,), check_trace=False)
        for pre_dispatch in (False, True):
            with pytest.raises(RuntimeError, match="trace"):
                make_fx(call, pre_dispatch=pre_dispatch)(x)


def test_gradients_forward_mode_transforms_and_traces_are_refused(monkeypatch):
    no_part_in("cpu", monkeypatch)


@gpu
def test_gradients_forward_mode_transforms_and_traces_are_refused_on_the_gpu(monkeypatch):
    assert fp6._ext is not None
    no_part_in(DEV, monkeypatch)


@gpu
@pytest.mark.parametrize("extension", [True, False])
def test_the_product_between_sort_and_sum(extension, monkeypatch):
    """A gradient of the tokens would end at the product: the call is refused, and works where the tokens are to get none; the sum's weights have theirs."""
    if not extension:
        monkeypatch.setattr(fp6, "_ext", None)
    E, T = 3, 5
    w = Weight(2, 64, 96, 32, True, E=E)
    index = torch.arange(2 * T, device=DEV).view(T, 2) % E
    x, weights = randn(3, T, 96).requires_grad_(), torch.rand(T, 2, device=DEV).requires_grad_()
    rows, plan = fp6.expert_sort(x, index, E)
    with pytest.raises(ValueError, match="no gradient"):
        fp6.int4_forward_native(rows, w.native, w.native_scales, plan)
    with torch.no_grad():
        y = fp6.int4_forward_native(rows, w.native, w.native_scales, plan)
    assert torch.equal(fp6.int4_forward_native(rows.detach(), w.native, w.native_scales, plan), y) and not y.requires_grad
    fp6.expert_combine(y, plan, weights).float().sum().backward()
    assert x.grad is None and weights.grad.shape == (T, 2)


# ---------------------------------------------------------------------------------------------------------------- sizes
def test_more_workgroups_than_a_grid_holds_are_refused():
    """A launch of 2^32 threads does nothing and says nothing."""
    from fp6_llm_amd import _lib
    L, p, SHAPE = _lib.lib(), 1 << 20, -2   # (an address that nothing reads: every call is refused before a launch)

    def cfg(kernel, M, N, dtype=0, offsets=None, E=1):
        return L.fp6mi_int4_linear_cfg(None, dtype, p, p, 128, 0, None, p, p, 0, -1, offsets, E, M, N, 128, p, kernel)
    for k in TILES:
        _, cols, row_tiles, _ = KERNELS[k]
        for M, N in ((16, cols << 23), (16 * row_tiles << 12, cols << 11)):
            assert all(cfg(k, M, N, dtype) == SHAPE for dtype in (0, 1)), k
        assert cfg(k, 16, 1 << 30, 0, p, 64) == SHAPE
    for k in STREAMS:
        assert cfg(k, 16, 65536 * 16) == SHAPE
    # the choice takes kernels that hold the problem, as long as there are any
    for N, of in ((65535 * 16, range(12)), (65536 * 16, TILES), (1 << 26, TILES), ((1 << 29) - 64, (10, 11)), ((1 << 29), (-2,)), (1 << 30, (-2,))):
        assert choice(16, N, 128) in of and choice(16, N, 128, "bf16") in of, N


@gpu
def test_more_bf16_rows_than_a_grid_has_workgroups():
    N = (1 << 24) + 3
    x, w = whole_numbers(Weight(1, 32, 64, 32, True, "bf16"), 2, 97)
    x = x.bfloat16().to(DEV)[torch.arange(N, device=DEV) * 5 % 97]
    assert choice(32, N, 64, "bf16", group=32) in TILES
    got = fp6.int4_forward_native(x, w.native, w.native_scales)
    want = (x[:97].double() @ w.w.t().to(DEV)).bfloat16()
    assert (x[:97].double() @ w.w.t().to(DEV)).abs().max() < 2 ** 24
    for first in range(0, N, 1 << 22):
        rows = torch.arange(first, min(N, first + (1 << 22)), device=DEV)
        assert torch.equal(got[first:first + (1 << 22)], want[rows % 97]), first


@gpu
def test_packing_more_than_a_grid_has_workgroups():
    """Blocks and scales of 65 matrices of 2^24 rows: the last one as by itself."""
    E, OC = 65, 1 << 24
    codes, scales = torch.empty(E, OC, 16, dtype=torch.uint8, device=DEV), torch.empty(E, OC, 1, dtype=torch.float16, device=DEV)
    for e in range(E):
        codes[e].random_(0, 256), scales[e].uniform_()
    native, native_scales = fp6.int4_pack_native(codes, scales, group=32)
    for e in (0, 15, 16, 31, 64):
        one, one_scales = fp6.int4_pack_native(codes[e], scales[e], group=32)
        assert torch.equal(native[e], one) and torch.equal(native_scales[e], one_scales), e
    del codes, scales, native, native_scales, one, one_scales
    torch.cuda.empty_cache()   # (100 GB)


# ---------------------------------------------------------------------------------------------------------------- views with a lazy negative sign
def test_packing_resolves_negative_views():
    w = Weight(3, 32, 96, 32, True, device="cpu")
    native, scales = fp6.int4_pack_native(w.codes, torch._neg_view(w.scales), w.zeros, 32)
    assert torch.equal(native, w.native) and torch.equal(scales[..., 0], -w.native_scales[..., 0]) and torch.equal(scales[..., 1], w.native_scales[..., 1])


@gpu
@pytest.mark.parametrize("N", [2, 100])
@pytest.mark.parametrize("extension", [True, False])
def test_negative_views(extension, N, monkeypatch):
    assert fp6._ext is not None
    if not extension:
        monkeypatch.setattr(fp6, "_ext", None)
    w = Weight(4, 64, 160, 32, False)
    x, b = randn(1, N, 160), randn(2, 64)
    want = fp6.int4_forward_native(x, w.native, w.native_scales, bias=b)
    neg = torch._neg_view
    assert torch.equal(fp6.int4_forward_native(neg(x), w.native, w.native_scales, bias=neg(b)), -want)
    assert torch.equal(fp6.int4_forward_native(x, w.native, neg(w.native_scales), bias=neg(b)), -want)
    assert torch.equal(fp6.int4_pack_native(w.codes, neg(w.scales), None, 32)[1], -w.native_scales)
    with pytest.raises(ValueError):
        fp6.int4_forward_native(x, w.native, w.native_scales, out=neg(torch.empty_like(want)))


# ---------------------------------------------------------------------------------------------------------------- outputs over inputs
@gpu
@pytest.mark.parametrize("extension", [True, False])
def test_outputs_over_inputs_are_refused(extension, monkeypatch):
    """Workgroups write rows of the output while others still read the input."""
    assert fp6._ext is not None
    if not extension:
        monkeypatch.setattr(fp6, "_ext", None)
    w = Weight(5, 64, 64, 32, True)
    both = randn(1, 41, 64)
    x = both[:40]
    want = fp6.int4_forward_native(x, w.native, w.native_scales)
    for out in (x, both[1:]):
        with pytest.raises(ValueError, match="memory of its own"):
            fp6.int4_forward_native(x, w.native, w.native_scales, out=out)
    beside = torch.empty(80, 64, dtype=torch.float16, device=DEV)
    beside[:40] = x
    assert torch.equal(fp6.int4_forward_native(beside[:40], w.native, w.native_scales, out=beside[40:]), want)
    strided = torch.empty(40, 128, dtype=torch.float16, device=DEV)   # (rows that are copied before the product)
    strided[:, ::2] = x
    assert torch.equal(fp6.int4_forward_native(strided[:, ::2], w.native, w.native_scales, out=strided.view(-1)[:40 * 64].view(40, 64)), want)


# ---------------------------------------------------------------------------------------------------------------- weights that have no codes
@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_refuses_what_has_no_codes(zeros):
    """A scale of infinity or NaN would make a group NaN whatever its codes; a float32 weight of 7 * 65504, or a range of 15 times that, still has a scale in fp16."""
    for dtype, value in ((torch.float32, float("inf")), (torch.float32, float("-inf")), (torch.float16, float("nan")), (torch.bfloat16, float("inf")), (torch.float32, 1.0e6), (torch.float32, 3.0e38)):
        w = torch.ones(2, 16, 64, dtype=dtype)
        w[1, 3, 40] = value
        if value == 1.0e6 and zeros:
            w[1, 3, 40] = 15 * 65600.0
        with pytest.raises(ValueError, match="infinities"):
            fp6.int4_quantize(w, 32, zeros)
    w = torch.ones(16, 64)
    w[3, 40] = 15 * 65504.0 if zeros else 7 * 65504.0
    codes, scales, z = fp6.int4_quantize(w, 32, zeros)
    assert scales[3, 1] == 65504 and codes[3, 20] & 15 == 15 and (z is None or z[3, 1] == 0)
