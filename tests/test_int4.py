"""Products with 4-bit integer weights and group scales against their definition in 64 bits.

Tolerances count roundings: half a step of fp16 is 2^-11 of the value (2^-25 below the normal numbers), of bf16 2^-8; products x * (q - z) are exact, and a float32 sum of n of them, the scaling of
each group and the sum over groups are off by at most (n + 2) * 2^-23 of the sum of all magnitudes, whatever the order and however the matrix unit rounds between them.  (In products of few bf16 rows the
terms are x * (128 + q) and -x * (128 + z), at most 143 each.)"""
import numpy as np
import pytest
import torch

import fp6_llm_amd as fp6
from fp6_llm_amd import _lib

DEV = "cuda:0"
gpu = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def d(t):
    return t.detach().cpu().double()


def within(got, want, tol, what=""):
    got = d(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s: got %s, want %s +- %s" % (
        what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), tol.expand_as(want)[bad][0].item())


class Weight:
    """Random codes, scales and zero points: as a checkpoint holds them, natively, and as numbers in 64 bits; E = 0: one matrix."""

    def __init__(self, seed, OC, IC, group=128, zeros=False, type="fp16", E=0, device=DEV):
        rng = np.random.default_rng(seed)
        lead = (E,) if E else ()
        groups = -(-IC // group)
        q = rng.integers(0, 16, lead + (OC, IC))
        z = rng.integers(0, 16, lead + (OC, groups)) if zeros else None
        scales = torch.from_numpy(np.exp(0.5 * rng.standard_normal(lead + (OC, groups))) / (5 * np.sqrt(IC))).to(TYPES[type])
        self.codes = torch.from_numpy((q[..., 0::2] | q[..., 1::2] << 4).astype(np.uint8)).to(device)
        self.scales, self.zeros = scales.to(device), None if z is None else torch.from_numpy(z.astype(np.uint8)).to(device)
        each = np.arange(IC) // group
        self.w = torch.from_numpy((q - (8 if z is None else z[..., each])).astype(np.float64)) * scales.double()[..., each]
        self.group, self.OC, self.IC, self.E, self.dtype = group, OC, IC, E, TYPES[type]
        self.native, self.native_scales = fp6.int4_pack_native(self.codes, self.scales, self.zeros, group)


def randn(seed, *shape, dtype=torch.float16, scale=1.0, device=DEV):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(device)


def product64(w, x, bias=None, extra=None):
    """x @ w^T + bias in 64 bits, and how far float32 sums may be from it (extra: of the 128 + q and -(128 + z) that stand for the codes and zero points of that weight)."""
    y, mag = d(x) @ w.t(), d(x).abs() @ w.abs().t()
    if extra is not None:
        mag = mag + d(x).abs() @ (2 * 143 * extra.scales.cpu().double().repeat_interleave(extra.group, 1)[:, :extra.IC]).t()
    if bias is not None:
        y, mag = y + d(bias), mag + d(bias).abs()
    return y, (w.shape[1] + 3) * 2.0 ** -23 * mag


def halves(p):
    p = p.reshape(p.shape[0], p.shape[1] // 32, 2, 16)
    return p[:, :, 0].flatten(1), p[:, :, 1].flatten(1)


def act64(act, g):
    if act == "silu":
        return g * torch.sigmoid(g)
    return torch.nn.functional.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")


def gated64(y, err, act, dtype):
    """act(gate) * up of pre-activations in pair order that are off by err.  The largest slopes are 1.1 (silu) and 1.13 (gelu); the functions are taken to 2^-18 of |g| at most."""
    (g, u), (eg, eu) = halves(y), halves(err)
    a = act64(act, g)
    ea = 1.13 * eg + 2.0 ** -18 * g.abs()
    h = a * u
    return h, (ea * u.abs() + eu * a.abs() + ea * eu) * (1 + HALF[dtype]) + HALF[dtype] * h.abs() + TINY[dtype]


def plain(y, err, dtype):
    return y, err * (1 + HALF[dtype]) + HALF[dtype] * y.abs() + TINY[dtype]


# ---------------------------------------------------------------------------------------------------------------- layout
def native_from_definition(codes, scales, zeros, group):
    """The native layout of one matrix, element by element from its description."""
    OC, IC = codes.shape[0], 2 * codes.shape[1]
    KB, each = -(-IC // 128), 128 if group % 128 == 0 else 64 if group % 64 == 0 else 32
    q = np.stack((codes & 15, codes >> 4), -1).reshape(OC, IC)
    w = np.zeros((OC // 16, KB, 256), dtype=np.uint32)
    s = np.zeros((OC // 16, KB, 16, 128 // each, 1 if zeros is None else 2), dtype=np.float32)
    nibble = [0, 4, 1, 5, 2, 6, 3, 7]
    for m in range(OC):
        for k in range(IC):
            step, quarter, j = k % 128 // 32, k % 32 // 8, k % 8
            w[m // 16, k // 128, (m % 16 + 16 * quarter) * 4 + step] |= np.uint32(q[m, k]) << np.uint32(4 * nibble[j])
            s[m // 16, k // 128, m % 16, k % 128 // each, 0] = scales[m, k // group]
            if zeros is not None:
                s[m // 16, k // 128, m % 16, k % 128 // each, 1] = zeros[m, k // group]
    return w, s


@pytest.mark.parametrize("OC,IC,group,zeros,type", [(16, 32, 32, True, "fp16"), (48, 320, 64, True, "bf16"), (32, 288, 96, False, "fp16"), (16, 512, 256, True, "bf16"), (32, 384, 128, False, "bf16"),
                                                     (16, 160, 1024, True, "fp16")])
def test_layout_is_what_its_description_says(OC, IC, group, zeros, type):
    w = Weight(OC + IC, OC, IC, group, zeros, type, device="cpu")
    want, scales = native_from_definition(w.codes.numpy(), w.scales.float().numpy(), None if w.zeros is None else w.zeros.numpy(), group)
    assert (w.native.numpy().view(np.uint32) == want).all()
    assert (w.native_scales.float().numpy() == scales).all()


def test_layout_of_experts_is_that_of_each():
    w = Weight(1, 32, 160, 64, True, E=3, device="cpu")
    for e in range(3):
        one, scales = fp6.int4_pack_native(w.codes[e], w.scales[e], w.zeros[e], 64)
        assert torch.equal(one, w.native[e]) and torch.equal(scales, w.native_scales[e])


@gpu
@pytest.mark.parametrize("OC,IC,group,zeros,type,E", [(16, 32, 32, True, "fp16", 0), (48, 320, 64, True, "bf16", 3), (272, 1056, 96, False, "fp16", 2), (64, 512, 256, True, "bf16", 0)])
def test_layout_made_on_the_gpu_is_that_of_the_host(OC, IC, group, zeros, type, E):
    a, b = Weight(5, OC, IC, group, zeros, type, E, "cpu"), Weight(5, OC, IC, group, zeros, type, E)
    assert torch.equal(a.native, b.native.cpu()) and torch.equal(a.native_scales, b.native_scales.cpu())
    apart = torch.cat((b.codes.new_zeros(3), b.codes.flatten()))[3:].view(b.codes.shape)   # (codes that begin between two 16-byte boundaries)
    native, scales = fp6.int4_pack_native(apart, b.scales, b.zeros, group)
    assert torch.equal(native, b.native) and torch.equal(scales, b.native_scales)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantizer_is_off_by_half_a_step(zeros, dtype):
    w = randn(3, 2, 48, 200, dtype=dtype, device="cpu") + (0.5 if zeros else 0.0)
    w[0, 3], w[0, 4, :64] = 0, 0.25
    codes, scales, z = fp6.int4_quantize(w, 64, zeros)
    assert codes.shape == (2, 48, 100) and scales.shape == (2, 48, 4) and (z is not None) == zeros
    assert scales.dtype == (torch.float16 if dtype == torch.float32 else dtype)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    each = torch.arange(200) // 64
    got = (q - (8 if z is None else z.double()[..., each])) * scales.double()[..., each]
    # half a step, another for a zero point that was rounded (its range ends half a step off), and 15 steps' share of the scale's own rounding
    step = scales.double()[..., each]
    assert ((got - w.double()).abs() <= step * (0.5 + 0.5 * zeros + 15 * HALF[scales.dtype]) + 2.0 ** -20).all()
    assert (got[0, 3] == 0).all()


# ---------------------------------------------------------------------------------------------------------------- one matrix
SHAPES = [  # OC, IC, N, group, zeros, type, bias
    (16, 32, 1, 32, False, "fp16", False), (16, 32, 3, 32, True, "bf16", True), (32, 128, 1, 128, True, "fp16", False), (48, 160, 2, 64, True, "bf16", False), (272, 1024, 1, 128, False, "fp16", True),
    (1040, 2080, 5, 32, True, "fp16", True), (512, 4576, 16, 32, False, "bf16", False), (256, 8192, 1, 64, True, "bf16", True), (4096, 256, 4, 128, False, "fp16", False), (336, 736, 15, 96, True, "fp16", False),
    (304, 1184, 17, 64, False, "fp16", True), (2064, 544, 31, 32, True, "bf16", False), (80, 4128, 33, 128, True, "fp16", False), (1024, 608, 48, 256, False, "bf16", True), (528, 1120, 64, 64, True, "fp16", False),
    (528, 1120, 65, 128, True, "bf16", True), (1296, 640, 100, 32, True, "fp16", True), (256, 2048, 129, 128, False, "fp16", False), (2320, 352, 200, 64, True, "bf16", False), (544, 1376, 300, 32, False, "bf16", True),
    (1072, 992, 513, 128, True, "fp16", True), (16, 96, 777, 32, True, "fp16", False), (4112, 416, 1030, 64, False, "fp16", False), (336, 128, 2500, 128, True, "bf16", False), (512, 11008, 20, 128, True, "fp16", False),
    (256, 28672, 2, 64, False, "fp16", False), (256, 28672, 70, 128, False, "bf16", False)]


@gpu
@pytest.mark.parametrize("OC,IC,N,group,zeros,type,bias", SHAPES)
def test_product(OC, IC, N, group, zeros, type, bias):
    w = Weight(OC + IC + N, OC, IC, group, zeros, type)
    x, b = randn(N, N, IC, dtype=w.dtype), randn(N + 1, OC, dtype=w.dtype) if bias else None
    y, err = product64(w.w, x, b, extra=w if type == "bf16" and choice(OC, N, IC, type) < 4 else None)
    within(fp6.int4_forward_native(x, w.native, w.native_scales, bias=b), *plain(y, err, w.dtype))
    within(fp6.int4_forward_native(x, w.native, w.native_scales, bias=b, out_dtype=torch.float32), *plain(y, err, torch.float32), "float32")


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("OC,IC,N,group,zeros,type,bias", [(32, 64, 1, 32, True, "fp16", True), (288, 1056, 7, 64, False, "bf16", True), (1120, 480, 40, 128, True, "fp16", False), (544, 2080, 150, 32, True, "bf16", True),
                                                            (2080, 256, 700, 128, False, "fp16", True)])
def test_gated_product(act, OC, IC, N, group, zeros, type, bias):
    w = Weight(OC + IC + N, OC, IC, group, zeros, type)
    x, b = randn(N, N, IC, dtype=w.dtype), randn(N + 1, OC, dtype=w.dtype) if bias else None
    y, err = product64(w.w, x, b)
    got = fp6.int4_forward_native(x, w.native, w.native_scales, activation=act, bias=b)
    assert got.dtype == w.dtype
    within(got, *gated64(y, err, act, w.dtype))
    within(fp6.int4_forward_native(x, w.native, w.native_scales, activation=act, bias=b, out_dtype=torch.float32), *gated64(y, err, act, torch.float32), "float32")


@gpu
@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("N", [1, 16, 40, 130])
def test_every_code_and_zero_point_is_exact(N, type):
    """One column at a time: y is x * s * (q - z) itself, with scales that are powers of two."""
    OC, IC = 256, 160
    q = (torch.arange(OC).unsqueeze(1) + torch.arange(IC)) % 16
    z = (torch.arange(OC).unsqueeze(1) // 16 + torch.arange(5)) % 16
    s = torch.exp2(((torch.arange(OC).unsqueeze(1) + torch.arange(5)) % 9 - 4).float()).to(TYPES[type])
    native, scales = fp6.int4_pack_native((q[:, 0::2] | q[:, 1::2] << 4).to(torch.uint8).to(DEV), s.to(DEV), z.to(torch.uint8).to(DEV), 32)
    columns = (torch.arange(N) * 37) % IC
    x = torch.zeros(N, IC)
    x[torch.arange(N), columns] = 1.5
    got = fp6.int4_forward_native(x.to(TYPES[type]).to(DEV), native, scales)
    each = torch.arange(IC) // 32
    want = (1.5 * (q - z[:, each]) * s.double()[:, each]).t()[columns]
    assert torch.equal(d(got), want)


@gpu
@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("N", [3, 20, 70, 300])
def test_rows_do_not_mix(N, type):
    """A NaN or an infinity in a row of the input reaches that row of the output alone."""
    w = Weight(9, 272, 672, 32, True, type)
    x = randn(4, N, 672, dtype=w.dtype)
    want = fp6.int4_forward_native(x, w.native, w.native_scales)
    x[N // 2, 5], x[N - 1, 671] = float("nan"), float("inf")
    got = fp6.int4_forward_native(x, w.native, w.native_scales)
    rest = [n for n in range(N) if n not in (N // 2, N - 1)]
    assert torch.equal(got[rest], want[rest]) and not got[N // 2].isfinite().any() and not got[N - 1].isfinite().any()


@gpu
@pytest.mark.parametrize("N", [1, 30, 300])
def test_scales_of_every_size(N):
    """Group sums are scaled in float32: neither the smallest fp16 scales nor the largest lose anything but what the output's type cannot hold."""
    w = Weight(2, 64, 256, 64, True)
    s = torch.exp2(torch.linspace(-24, 11, 256).round()).view(64, 4)   # (up to 15 * 8 * 64 * 2^11 in a group)
    native, scales = fp6.int4_pack_native(w.codes, s.half().to(DEV), w.zeros, 64)
    x = randn(6, N, 256)
    w64 = w.w / w.scales.cpu().double().repeat_interleave(64, 1) * s.double().repeat_interleave(64, 1)
    y, err = product64(w64, x)
    within(fp6.int4_forward_native(x, native, scales, out_dtype=torch.float32), *plain(y, err, torch.float32))


@gpu
@pytest.mark.parametrize("N", [3, 40])
@pytest.mark.parametrize("type", ["fp16", "bf16"])
def test_rows_longer_than_a_tile_takes(N, type):
    """More than 2^20 columns: offsets of 16 rows pass 2^25 bytes, and the kernels that stream weights take any number of rows."""
    w = Weight(3, 32, (1 << 20) + 160, 128, True, type)
    x = randn(4, N, w.IC, dtype=w.dtype)
    assert choice(32, N, w.IC, type) not in TILES
    y, err = product64(w.w, x, extra=w if type == "bf16" else None)
    within(fp6.int4_forward_native(x, w.native, w.native_scales), *plain(y, err, w.dtype))


@gpu
def test_no_rows_give_no_rows():
    w = Weight(1, 32, 64, 32)
    got = fp6.int4_forward_native(torch.empty(0, 64, dtype=torch.float16, device=DEV), w.native, w.native_scales)
    assert got.shape == (0, 32) and got.dtype == torch.float16


@gpu
def test_strided_rows_given_outputs_and_another_stream():
    w = Weight(11, 272, 480, 32, True)
    wide = randn(1, 60, 960)
    x = wide[:, 480:]
    want = fp6.int4_forward_native(x.contiguous(), w.native, w.native_scales)
    out = torch.full((60, 272), float("nan"), dtype=torch.float16, device=DEV)
    assert fp6.int4_forward_native(x, w.native, w.native_scales, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp6.int4_forward_native(x, w.native, w.native_scales)
    side.synchronize()
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("N", [1, 40, 200])
def test_captured_product_replays_to_the_eager_results(N):
    w = Weight(12, 544, 736, 32, True, "bf16")
    x = randn(1, N, 736, dtype=w.dtype)
    out = fp6.int4_forward_native(x, w.native, w.native_scales, activation="silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fp6.int4_forward_native(x, w.native, w.native_scales, activation="silu")
    for seed in range(2, 6):
        x.copy_(randn(seed, N, 736, dtype=w.dtype))
        out = fp6.int4_forward_native(x, w.native, w.native_scales, activation="silu")
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


@gpu
@pytest.mark.parametrize("N", [1, 50, 300])
def test_calls_without_the_extension(N, monkeypatch):
    assert fp6._ext is not None
    w = Weight(13, 288, 672, 64, True)
    x, b = randn(2, N, 672), randn(3, 288)
    args = [dict(), dict(bias=b), dict(activation="gelu", bias=b), dict(out_dtype=torch.float32)]
    first = [fp6.int4_forward_native(x, w.native, w.native_scales, **a) for a in args]
    monkeypatch.setattr(fp6, "_ext", None)
    for a, want in zip(args, first):
        got = fp6.int4_forward_native(x, w.native, w.native_scales, **a)
        assert got.dtype == want.dtype and torch.equal(got, want)


# ---------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_packer():
    codes, scales = torch.zeros(32, 32, dtype=torch.uint8), torch.ones(32, 2, dtype=torch.float16)
    ok = fp6.int4_pack_native(codes, scales, None, 32)
    assert ok[0].shape == (2, 1, 256)
    for bad in (dict(codes=codes.int()), dict(codes=codes[0]), dict(codes=codes[:20]), dict(codes=codes[:, :24]), dict(group=0), dict(group=48), dict(group=-32), dict(group=128), dict(scales=scales.float()),
                dict(scales=scales[:16]), dict(zeros=torch.zeros(32, 2, dtype=torch.int32)), dict(zeros=torch.zeros(32, 1, dtype=torch.uint8)), dict(codes=torch.zeros(0, 32, 32, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            fp6.int4_pack_native(**{**dict(codes=codes, scales=scales, zeros=None, group=32), **bad})
    for bad in (dict(weight=torch.zeros(4, 5)), dict(weight=torch.zeros(64)), dict(weight=torch.zeros(4, 64, dtype=torch.int32)), dict(group=40), dict(group=0)):
        with pytest.raises(ValueError):
            fp6.int4_quantize(**{**dict(weight=torch.zeros(4, 64)), **bad})


def test_refusals_of_the_c_abi():
    L, p = _lib.lib(), 1 << 20   # (an address that nothing reads: every call is refused before a launch)
    SHAPE, NULL, ALIGN, ACT, TYPE = -2, -3, -6, -9, -10
    assert L.fp6mi_int4_weight_bytes(1, 24, 64) == 0 and L.fp6mi_int4_weight_bytes(1, 16, 48) == 0 and L.fp6mi_int4_weight_bytes(0, 16, 64) == 0 and L.fp6mi_int4_weight_bytes(3, 32, 160) == 3 * 2 * 2 * 1024
    assert L.fp6mi_int4_scale_bytes(1, 16, 64, 40, 0) == 0 and L.fp6mi_int4_scale_bytes(2, 16, 160, 96, 1) == 2 * 16 * 2 * 4 * 4

    def linear(dtype=0, W=p, S=p, group=64, zeros=0, bias=None, X=p, Y=p, f32=0, act=-1, offsets=None, E=1, M=32, N=2, K=64, ws=None):
        return L.fp6mi_int4_linear(None, dtype, W, S, group, zeros, bias, X, Y, f32, act, offsets, E, M, N, K, ws)
    assert linear(dtype=2) == TYPE and linear(dtype=-1) == TYPE
    for bad in (dict(group=96), dict(group=0), dict(M=24), dict(M=0), dict(K=48), dict(K=0), dict(E=2), dict(E=0), dict(E=2000, offsets=p), dict(act=0, M=48), dict(N=(1 << 30) + 1), dict(M=1 << 25), dict(K=1 << 25)):
        assert linear(**bad) == SHAPE, bad
    assert linear(act=3) == ACT
    for name in ("W", "S", "X", "Y"):
        assert linear(**{name: None}) == NULL and linear(**{name: p + 8}) == ALIGN
    assert linear(bias=p + 1) == ALIGN and linear(offsets=p + 2) == ALIGN
    assert linear(N=0, X=None, Y=None) == 0 and linear(dtype=1, M=8192, K=8192, N=500) == -4 and linear(ws=p + 8) == ALIGN
    assert L.fp6mi_int4_workspace_bytes(0, 64, 1, 0, 32, 500, 64, 0, 8) == 0 and L.fp6mi_int4_workspace_bytes(1, 64, 1, 0, 32, 500, 64, 0, 8) == 2000 + 500 * 128
    assert L.fp6mi_int4_workspace_bytes(1, 64, 1, 0, 32, 500, 64, 0, 3) == 0 and L.fp6mi_int4_workspace_bytes(1, 64, 1, 0, 32, 500, 64, 0, 12) == 0 and L.fp6mi_int4_workspace_bytes(1, 64, 1, 0, 32, 0, 64, 0, 8) == 0 and L.fp6mi_int4_workspace_bytes(1, 96, 1, 0, 32, 500, 64, 0, 8) == 0

    def cfg(kernel, act=-1, K=64):
        return L.fp6mi_int4_linear_cfg(None, 1, p, p, 64, 0, None, p, p, 0, act, None, 1, 32, 2, K, None, kernel)
    assert cfg(12) == SHAPE and all(cfg(k, act=0) == SHAPE for k in UNPAIRED) and all(cfg(k, K=(1 << 20) + 32) == SHAPE and cfg(k) == (SHAPE if k == 10 else -4) for k in TILES)   # (10: groups of 128)
    assert L.fp6mi_int4_pack(p, p, p, p, None, 2, 1, 16, 64, 64) == TYPE and L.fp6mi_int4_pack(p, p, p, None, None, 0, 1, 16, 64, 64) == NULL
    assert L.fp6mi_int4_pack_gpu(None, p, p, p, p, None, 0, 1, 16, 64, 33) == SHAPE and L.fp6mi_int4_pack_gpu(None, p + 4, p, p, p, None, 0, 1, 16, 64, 64) == ALIGN


def refusals(x, w, monkeypatch):
    ok = dict(in_feats=x, native_weight=w.native, native_scales=w.native_scales)
    plan = fp6.experts.ExpertPlan(torch.zeros(7, dtype=torch.int32, device=x.device), 1, 2, 2)
    cases = [dict(in_feats=x.float()), dict(in_feats=x.bfloat16()), dict(in_feats=x[0]), dict(in_feats=x[:, :32]), dict(in_feats=x[:, :40]), dict(in_feats=x.cpu()), dict(native_weight=w.native.float()),
             dict(native_weight=w.native[:1]), dict(native_weight=w.native[..., :128]), dict(native_scales=w.native_scales[..., 0]), dict(native_scales=w.native_scales.float()), dict(activation="relu"),
             dict(activation=3), dict(out_dtype=torch.bfloat16), dict(out_dtype=torch.float64), dict(out=torch.empty(2, 32, device=x.device)), dict(out=torch.empty(2, 31, dtype=torch.float16, device=x.device)),
             dict(bias=torch.zeros(31, dtype=torch.float16, device=x.device)), dict(bias=torch.zeros(32, device=x.device)), dict(plan=plan)]
    for ext in (fp6._ext, None):
        monkeypatch.setattr(fp6, "_ext", ext)
        for bad in cases:
            if bad.get("in_feats") is not None and bad["in_feats"].device.type == "cpu" and x.device.type == "cpu":
                bad = dict(in_feats=x)
            with pytest.raises(ValueError):
                fp6.int4_forward_native(**{**ok, **bad})


def test_refusals_of_the_function(monkeypatch):
    """On the host every call is refused; that none of them gets to a launch is what counts."""
    w = Weight(1, 32, 160, 32, True, device="cpu")
    refusals(randn(1, 2, 160, device="cpu"), w, monkeypatch)


@gpu
def test_refusals_of_the_function_on_the_gpu(monkeypatch):
    w = Weight(1, 32, 160, 32, True)
    refusals(randn(1, 2, 160), w, monkeypatch)


# ---------------------------------------------------------------------------------------------------------------- the kernels by number
KERNELS = [(0, 16, 1, 16), (0, 16, 2, 8), (0, 16, 3, 8), (0, 16, 4, 8), (0, 16, 4, 4),
           (1, 32, 3, 4), (1, 32, 4, 4), (1, 32, 6, 4), (1, 32, 8, 4), (1, 32, 8, 2), (1, 64, 8, 2), (1, 64, 16, 1)]   # tiles, rows of X, row tiles, parts of K
TILES, UNPAIRED = range(5, 12), (0, 2, 5, 7)   # (those without a gated product: a wavefront's row tiles are not pairs)


def choice(OC, N, IC, type="fp16", E=0, gated=False, group=128):
    import ctypes
    shape = (ctypes.c_int * 4)()
    k = _lib.lib().fp6mi_int4_query_kernel(0 if type == "fp16" else 1, group, E or 1, E > 0, OC, N, IC, gated, shape)
    assert k < 0 or tuple(shape) == KERNELS[k]
    return k


def test_every_kernel_is_asked_for():
    """Each of the kernels is the choice somewhere in the range that is used."""
    for gated in (False, True):
        found = {choice(OC, N, IC, gated=gated) for OC in (256, 1008, 2064, 4112, 8208, 14352, 28688) for IC in (288, 1056, 2080, 4192, 8192, 11040, 28672) for N in (1, 8, 14, 20, 33, 61, 75, 125, 193, 260, 400, 521, 800, 2000)}
        assert found == set(range(len(KERNELS))) - set(UNPAIRED if gated else ())


def test_choices_are_in_range():
    for type in ("fp16", "bf16"):
        for E in (0, 1, 7, 128, 1024):
            for OC in (32, 4128, 1 << 20):
                for N in (1, 100, 5000, 1 << 22, 1 << 30):
                    for IC in (32, 4128, 1 << 21):
                        for gated in (False, True):
                            k = choice(OC, N, IC, type, E, gated, 64)
                            assert k == -2 or (0 <= k < len(KERNELS) and (k not in TILES or IC <= 1 << 20) and (k not in UNPAIRED or not gated) and k != 10)


def by_kernel(kernel, w, x, bias=None, act=-1, f32=False, plan=None):
    """The product by one kernel, into rows with others behind them that have to stay as they are."""
    L, s = _lib.lib(), w.native_scales
    N, E, type = x.shape[0], w.E or 1, 0 if w.dtype == torch.float16 else 1
    cols = w.OC // 2 if act >= 0 else w.OC
    whole = torch.full((N + 3, cols), 7.0, dtype=torch.float32 if f32 else w.dtype, device=DEV)
    need = L.fp6mi_int4_workspace_bytes(type, 128 // s.shape[-2], E, plan is not None, w.OC, N, w.IC, act >= 0, kernel)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    rc = L.fp6mi_int4_linear_cfg(torch.cuda.current_stream().cuda_stream, type, w.native.data_ptr(), s.data_ptr(), 128 // s.shape[-2], s.shape[-1] - 1, None if bias is None else bias.data_ptr(), x.data_ptr(),
                                 whole.data_ptr(), f32, act, None if plan is None else plan.offsets.data_ptr(), E, w.OC, N, w.IC, ws.data_ptr() if need else None, kernel)
    assert rc == 0, rc
    assert (whole[N:] == 7.0).all()
    return whole[:N]


@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (32, False), (64, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("type", ["fp16", "bf16"])
@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_every_kernel_with_every_layout(kernel, type, group, zeros):
    """Row tiles that do not fill a workgroup, one to five parts of K, the last block cut, rows of X at the borders of a tile; sums as they are, rounded, with a bias, gated."""
    if kernel == 10 and group != 128:
        pytest.skip("this kernel has groups of 128 only")
    cols = KERNELS[kernel][1]
    for OC, IC, N in ((48, 32, 1), (272, 96, cols), (96, 1184, cols + 1), (1056, 608, 2 * cols - 1), (32, 4128, 3), (288, 2048, 3 * cols + 5)):
        w = Weight(OC + N + kernel, OC, IC, group, zeros, type)
        x, b = randn(N, N, IC, dtype=w.dtype), randn(N + 1, OC, dtype=w.dtype)
        # (in few bf16 rows -(128 + z) and 128 + q stand for q - z)
        y, err = product64(w.w, x, b, extra=w if type == "bf16" and kernel not in TILES else None)
        within(by_kernel(kernel, w, x, b), *plain(y, err, w.dtype), "%s" % ((OC, IC, N),))
        within(by_kernel(kernel, w, x, b, f32=True), *plain(y, err, torch.float32), "float32 %s" % ((OC, IC, N),))
        if kernel not in UNPAIRED and OC % 32 == 0:
            within(by_kernel(kernel, w, x, b, act=1), *gated64(y, err, "gelu", w.dtype), "gated %s" % ((OC, IC, N),))


@gpu
@pytest.mark.parametrize("kernel", TILES)
def test_bf16_rows_of_every_size_in_tiles(kernel):
    """Rows of bf16 are multiplied as fp16 with a power of two each: magnitudes from the smallest to the largest, zeros, infinities and NaN."""
    w = Weight(5, 64, 160, 128 if kernel == 10 else 32, True, "bf16")
    x = randn(3, 12, 160, dtype=torch.float32, device="cpu")
    x *= torch.exp2(torch.tensor([0, -60, 60, -126, 100, -133, 10, 0, 0, 0, 0, 0])).unsqueeze(1)
    x[7] = 0
    x[8, 3], x[9, 5], x[10, 0], x[11, 1:] = float("inf"), float("nan"), 2.0 ** 30, 2.0 ** -20
    x[11, 0] = 2.0 ** 19
    x = x.bfloat16().to(DEV)
    got = by_kernel(kernel, w, x, f32=True)
    fine = [n for n in range(12) if n not in (8, 9)]
    y, err = product64(w.w, x[fine])
    # (values below 2^-32 of their row's largest: 2^-40 of that, times the sum of the weights)
    lost = 2.0 ** -40 * d(x[fine]).abs().amax(1, keepdim=True) * w.w.abs().sum(1)
    within(got[fine], y, err * (1 + 2.0 ** -24) + lost + 2.0 ** -24 * y.abs() + 2.0 ** -149)
    k = w.w[:, 3]
    assert torch.equal(torch.isinf(d(got[8])), k != 0) and torch.equal(d(got[8])[k != 0] > 0, k[k != 0] > 0) and got[9].isnan().all()


def test_waits_of_the_tile_kernels_cover_the_transfers(tmp_path):
    """int4_tile waits for its transfers to LDS by the number of loads that come behind them, which the compiler issues: in the compiled loop, as many stand between a transfer and its wait."""
    import os
    import re
    from concurrent.futures import ThreadPoolExecutor
    from fp6_llm_amd import build
    try:
        build.hipcc_path()
    except RuntimeError:
        pytest.skip("no compiler here")
    units = [u for u in build.UNITS if u[0] == "fp6mi_int4.hip"]

    def kernels_of(unit):
        src, obj, flags = unit
        out = str(tmp_path / (obj + ".s"))
        build._hipcc(["--cuda-device-only", "-S", os.path.join(build.HERE, "csrc", src), "-o", out] + flags, out, False)
        with open(out) as f:
            return re.findall(r"^(_ZN\w*int4_tile\w*):[^\n]*\n(.*?)s_endpgm", f.read(), re.S | re.M)
    with ThreadPoolExecutor(len(units)) as pool:
        kernels = [k for ks in pool.map(kernels_of, units) for k in ks]
    assert len(kernels) == 12 * 6 + 4   # (kernels 5 to 11, of which 10 has groups of 128 only)
    vector = re.compile(r"(buffer|global|scratch|flat)_(load|store|atomic)")
    for name, text in kernels:
        loop = max(re.split(r"\n\.LBB[^\n]*:", text), key=lambda b: b.count("v_mfma"))
        ops = [line.split(";")[0].strip() for line in loop.splitlines()]
        waits = [i for i, op in enumerate(ops) if op == "s_barrier"]
        assert len(waits) == 2, name   # (two blocks to a turn of the loop)
        for at in waits:
            n = int(re.fullmatch(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)", ops[at - 1]).group(1))
            behind = 0
            for op in ops[:at][::-1] + ops[at:][::-1]:   # (backwards, around the loop)
                if op.endswith(" lds"):
                    break
                behind += bool(vector.match(op))
            assert n <= behind < 64, (name, n, behind)
