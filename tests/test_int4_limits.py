"""Products with 4-bit integer weights at the ends of their ranges: values, sizes, and calls that they have no part in."""
import pytest
import torch

import fp6_llm_amd as fp6
from test_int4 import DEV, KERNELS, TILES, TYPES, Weight, by_kernel, choice, d, gpu, randn

STREAMS = [k for k in range(len(KERNELS)) if k not in TILES]


def whole_numbers(w, seed, N):
    """Rows of -1, 0 and 1 for a weight whose scales become 1 and 2: sums of whole numbers, which float32 holds in any order, and the same in 64 bits."""
    s = torch.exp2(torch.randint(0, 2, w.scales.shape, generator=torch.Generator().manual_seed(seed)).double())
    each = torch.arange(w.IC) // w.group
    old = w.scales.cpu().double()
    w.w = (w.w / old[..., each]).round() * s[..., each]
    w.scales = s.to(w.dtype).to(DEV)
    w.native, w.native_scales = fp6.int4_pack_native(w.codes, w.scales, w.zeros, w.group)
    x = torch.randint(-1, 2, (N, w.IC), generator=torch.Generator().manual_seed(seed + 1)).double()
    return x, w


# ---------------------------------------------------------------------------------------------------------------- infinities and large values
@gpu
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("kernel", STREAMS)
def test_bf16_rows_of_every_size_in_the_stream_kernels(kernel, group, zeros):
    """These multiply 128 + q, which leaves float32's range before q - z does: all that float32 sums of the weights' own products can hold comes out, and infinities as the definition has them.  Rows of
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
@pytest.mark.parametrize("act", [None, "silu"])
def test_an_infinity_in_a_bf16_row_does_not_depend_on_how_many_rows_there_are(act):
    w = Weight(6, 4096, 512, 128, True, "bf16")
    x = randn(1, 2048, 512, dtype=torch.bfloat16)
    x[0, 7], x[0, 300] = float("inf"), 2.0 ** 122
    assert choice(4096, 1, 512, "bf16", gated=act is not None) in STREAMS and choice(4096, 2048, 512, "bf16", gated=act is not None) in TILES
    few, many = (fp6.int4_forward_native(x[:n], w.native, w.native_scales, activation=act, out_dtype=torch.float32)[0] for n in (1, 2048))
    assert torch.equal(few.isnan(), many.isnan()) and torch.equal(few[~few.isnan()], many[~many.isnan()]) and few.isinf().any()
