"""Timed cases of the operators around the FPx linear layer: the gated feed-forward block (forward; forward and backward), the input
gradient of a linear layer, and low-rank adapters of many requests beside a shared projection.

`own` chooses between the package's entry points and a plain form in elementary torch operations, 32 bits throughout.  Weights are given as what the
codes stand for (value times the power of two of its group) and a factor per row; the package's side holds them in its native layout, as a program that has loaded a
checkpoint does.  M = weight rows, K = input features, N = tokens, F = M / 2 outputs of a gated block, R = rank.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
FORMATS = ((3, 2), (2, 2), (2, 3), (2, 1))
MAX_FLOPS = 2 * 2 * 28672 * 8192 * 2048   # the largest listed case


def _gated(name, E, Mb, F, K, N, act="silu", groups=False, bias=False, train=False):
    return {"name": name, "kind": "gated_train" if train else "gated", "E": E, "Mb": Mb, "F": F, "K": K, "N": N, "act": act, "groups": groups, "bias": bias}


def _grad(name, E, Mb, M, K, N, groups=False):
    return {"name": name, "kind": "grad", "E": E, "Mb": Mb, "M": M, "K": K, "N": N, "groups": groups}


def _adapters(name, E, Mb, M, K, N, R, slots, requests, bias=False, groups=False):
    return {"name": name, "kind": "adapters", "E": E, "Mb": Mb, "M": M, "K": K, "N": N, "R": R, "slots": slots, "requests": requests, "bias": bias, "groups": groups}


def listed():
    return [
        # one token through the feed-forward block of a small model: the call's own latency counts
        _gated("gated_11008x4096_n1", 3, 2, 11008, 4096, 1),
        # a serving batch of a large model with 4-bit weights and group exponents
        _gated("gated_28672x8192_n16_e2m1_groups", 2, 1, 28672, 8192, 16, groups=True),
        # a scheduler's odd batch: too many tokens for the small-batch kernels, too few for the large ones; 5-bit weights
        _gated("gated_11008x4096_n72_e2m2", 2, 2, 11008, 4096, 72),
        # a ragged prompt on a ragged matrix (K cuts the last block of 256 columns), another activation, biases
        _gated("gated_2304x4544_n777_e2m3", 2, 3, 2304, 4544, 777, act="gelu_tanh", groups=True, bias=True),
        # a prompt chunk of a large model: the largest case
        _gated("gated_28672x8192_n2048", 3, 2, 28672, 8192, 2048),
        # a training step of the block over a short and over a long sequence: output, gradient of the input and of the pre-activations
        _gated("gated_train_11008x4096_n512", 3, 2, 11008, 4096, 512, train=True),
        _gated("gated_train_11008x4096_n4096", 3, 2, 11008, 4096, 4096, train=True),
        # a gradient through few tokens (a soft prompt), through a ragged batch, and through a long sequence
        _grad("grad_4096x4096_n8", 3, 2, 4096, 4096, 8),
        _grad("grad_4608x4544_n333_e2m2_groups", 2, 2, 4608, 4544, 333, groups=True),
        _grad("grad_8192x8192_n4096", 3, 2, 8192, 8192, 4096),
        # a decode step of 32 requests, each with an adapter of its own or none; a long batch of prompts of several requests
        _adapters("adapters_4096x4096_n32_r16", 3, 2, 4096, 4096, 32, 16, 64, 32),
        _adapters("adapters_10240x8192_n2048_r64", 3, 2, 10240, 8192, 2048, 64, 16, 11, bias=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    E, Mb = rng.choice(FORMATS)
    groups = rng.random() < 0.3
    K = min(8192, max(1024, 64 * round(log(1024, 8192) / 64)))
    N = log(1, 4096)
    kind = rng.choice(("gated", "gated_train", "grad", "adapters"))
    while True:
        if kind.startswith("gated"):
            F = 256 * rng.randint(4, 112)
            work_ = (6 if kind == "gated_train" else 2) * N * 2 * F * K
            case = _gated("", E, Mb, F, K, N, rng.choice(("silu", "gelu", "gelu_tanh")), groups, rng.random() < 0.3, kind == "gated_train")
        else:
            M = 256 * rng.randint(4, 112)
            work_ = 2 * N * M * K
            if kind == "grad":
                case = _grad("", E, Mb, M, K, N, groups)
            else:
                R, slots = 8 * rng.randint(1, 16), rng.randint(1, 64)
                case = _adapters("", E, Mb, M, K, N, R, slots, rng.randint(1, max(1, min(N, 64))), rng.random() < 0.3, groups)
        if work_ <= MAX_FLOPS // 2:
            del case["name"]
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _magnitudes(E, Mb):
    bias = (1 << (E - 1)) - 1
    return [2.0 ** (1 - bias) * m / (1 << Mb) if e == 0 else 2.0 ** (e - bias) * (1 + m / (1 << Mb)) for e in range(1 << E) for m in range(1 << Mb)]


def _weights(g, E, Mb, M, K, groups):
    """values [M, K] fp16 (exact) and scales [M] fp16 of a weight that was quantized with one scale a row and, with groups, a power of two for every 128
    columns: about normal values, in every row one of the largest magnitude."""
    mags = torch.tensor(_magnitudes(E, Mb), device=DEVICE, dtype=torch.float32)
    top = mags[-1]
    v = torch.empty(M, K, device=DEVICE, dtype=torch.float16)
    steps = (mags[1:] + mags[:-1]) / 2
    for r in range(0, M, 4096):   # (in pieces: 32-bit noise for the whole of a large matrix takes gigabytes)
        z = torch.randn(min(4096, M - r), K, generator=g, device=DEVICE) * (top / 4.2)
        v[r:r + z.shape[0]] = mags[torch.bucketize(z.abs(), steps)].copysign(z).half()
    at = torch.randint(0, K, (M, 1), generator=g, device=DEVICE)
    if groups:
        k = torch.randint(-3, 1, (M, (K + 127) // 128), generator=g, device=DEVICE)
        k.scatter_(1, at // 128, 0)
        for j in range(k.shape[1]):
            v[:, 128 * j:128 * j + 128] *= torch.exp2(k[:, j:j + 1].float()).half()
    v.scatter_(1, at, top.half().expand(M, 1))
    rms = top / 4.2
    scales = (torch.exp(0.2 * torch.randn(M, generator=g, device=DEVICE)) / (rms * math.sqrt(K))).half()
    return v, scales


def _native(case, v, scales):
    """The package's side: quantized on the GPU from the float weights, which gives back these very values and scales."""
    import fp6_llm_amd as fp6
    w = torch.empty(v.shape, device=DEVICE, dtype=torch.float32)
    for r in range(0, v.shape[0], 4096):
        w[r:r + 4096] = v[r:r + 4096].float() * scales[r:r + 4096].float()[:, None]
    out = fp6.weight_quantize_native_cuda(case["E"], case["Mb"], w, case["groups"])
    return out if case["groups"] else out + (None,)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    N, K = case["N"], case["K"]
    M = case.get("M", 2 * case.get("F", 0))
    d = {}
    d["v"], d["scales"] = _weights(g, case["E"], case["Mb"], M, K, case["groups"])
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)   # noqa: E731
    d["bias"] = (0.1 * randn(M)).half() if case.get("bias") else None
    if case["kind"] != "grad":
        d["x"] = randn(N, K).half()
    if case["kind"] == "grad":
        d["dy"] = (0.05 * randn(N, M)).half()
    if case["kind"] == "gated_train":
        d["dh"] = (0.05 * randn(N, M // 2)).half()
    if case["kind"] == "adapters":
        R, S = case["R"], case["slots"]
        d["a"] = (randn(S, R, K) / math.sqrt(K)).half()
        d["b"] = (0.3 * randn(S, M, R) / math.sqrt(R)).half()
        d["s"] = torch.exp2(torch.randint(-1, 2, (S,), generator=g, device=DEVICE).float())
        # a batch of requests one behind the other (of one token each in a decode step), an eighth of them without an adapter
        slot = torch.randint(0, S, (case["requests"],), generator=g, device=DEVICE)
        slot[torch.rand(case["requests"], generator=g, device=DEVICE) < 0.125] = -1
        cuts = torch.rand(N, generator=g, device=DEVICE).argsort()[:case["requests"]].sort().values
        if case["requests"] > 0:
            cuts[0] = 0
        which = torch.bucketize(torch.arange(N, device=DEVICE), cuts, right=True) - 1
        d["index"] = slot[which].int()
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": case, **d}
    if own:
        state["w"], state["sc"], state["exps"] = _native(case, d["v"], d["scales"])
        del state["v"], state["scales"]
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def _act(act, g):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def _act_grad(act, g):
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * math.sqrt(0.5 / math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _halves(p):
    """Pair order (16 gate rows, the same 16 of up, ...) -> gate and up."""
    p = p.view(p.shape[0], -1, 2, 16)
    return p[:, :, 0].flatten(1), p[:, :, 1].flatten(1)


def _pairs(g, u):
    return torch.stack((g.view(g.shape[0], -1, 16), u.view(u.shape[0], -1, 16)), 2).flatten(1)


def _product(x, v, scales, bias):
    y = (x.float() @ v.float().t()) * scales.float()
    return y if bias is None else y + bias.float()


def _plain(s):
    c = s["case"]
    if c["kind"] == "grad":
        return ((s["dy"].float() * s["scales"].float()) @ s["v"].float()).half()
    y = _product(s["x"], s["v"], s["scales"], s["bias"])
    if c["kind"] == "adapters":
        x, idx = s["x"].float(), s["index"].long()
        for slot in torch.unique(idx).tolist():
            if slot >= 0:
                rows = (idx == slot).nonzero()[:, 0]
                y[rows] += s["s"][slot] * ((x[rows] @ s["a"][slot].float().t()) @ s["b"][slot].float().t())
        return y.half()
    g, u = _halves(y)
    a = _act(c["act"], g)
    h = (a * u).half()
    if c["kind"] == "gated":
        return h
    dh = s["dh"].float()
    dp = _pairs(dh * u * _act_grad(c["act"], g), dh * a)
    return {"out": h, "grad_in": ((dp * s["scales"].float()) @ s["v"].float()).half(), "grad_preact": dp.half()}


def _own(s):
    import fp6_llm_amd as fp6
    c = s["case"]
    E, Mb, w, sc, ge = c["E"], c["Mb"], s["w"], s["sc"], s["exps"]
    if c["kind"] == "grad":
        return fp6.linear_input_grad_native(E, Mb, s["dy"], w, sc, c["K"], group_exps=ge)
    if c["kind"] == "adapters":
        return fp6.adapter_forward_native(E, Mb, s["x"], w, sc, c["M"], s["a"], s["b"], s["s"], s["index"], group_exps=ge, bias=s["bias"])
    M = 2 * c["F"]
    if c["kind"] == "gated":
        return fp6.gated_forward_native(E, Mb, s["x"], w, sc, M, c["act"], group_exps=ge, bias=s["bias"])
    preact = torch.empty(c["N"], M, device=DEVICE)
    h = fp6.gated_forward_native(E, Mb, s["x"], w, sc, M, c["act"], preact=preact, group_exps=ge, bias=s["bias"])
    dx, dp = fp6.gated_backward_native(E, Mb, s["dh"], preact, w, sc, c["K"], c["act"], group_exps=ge)
    return {"out": h, "grad_in": dx, "grad_preact": dp}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------- what a pass is measured against
def work(case):
    N, K = case["N"], case["K"]
    M = case.get("M", 2 * case.get("F", 0))
    weights = M * K * (1 + case["E"] + case["Mb"]) // 8 + 2 * M + (M * ((K + 127) // 128) if case["groups"] else 0) + (2 * M if case.get("bias") else 0)
    flops = 2 * N * M * K
    if case["kind"] == "grad":
        return {"bytes": weights + 2 * N * (M + K), "flops": flops}
    if case["kind"] == "gated":
        return {"bytes": weights + 2 * N * (K + M // 2), "flops": flops}
    if case["kind"] == "gated_train":   # forward, then backward: x and dh in, h, dx and the gradient of the pre-activations out
        return {"bytes": weights + 2 * N * (2 * K + 2 * (M // 2) + M), "flops": 2 * flops}
    used = min(case["requests"], case["slots"])
    return {"bytes": weights + 2 * N * (K + M) + 2 * used * case["R"] * (K + M) + 4 * N, "flops": flops + 2 * N * case["R"] * (K + M)}


def exact(case, seed):
    """The definitions in 64 bits, a slice of output columns at a time."""
    d = _inputs(case, seed)
    W = lambda lo, hi: d["v"][lo:hi].double() * d["scales"][lo:hi].double().unsqueeze(1)   # noqa: E731
    M, K = d["v"].shape
    N = case["N"]
    if case["kind"] == "grad":
        dx = torch.zeros(N, K, dtype=torch.float64, device=DEVICE)
        for r in range(0, M, 4096):
            dx.addmm_(d["dy"][:, r:r + 4096].double(), W(r, r + 4096))
        return dx
    x = d["x"].double()
    y = torch.empty(N, M, dtype=torch.float64, device=DEVICE)
    for r in range(0, M, 4096):
        y[:, r:r + 4096] = torch.mm(x, W(r, r + 4096).t())
    if d["bias"] is not None:
        y += d["bias"].double()
    if case["kind"] == "adapters":
        for n, slot in enumerate(d["index"].tolist()):
            if slot >= 0:
                y[n] += d["s"][slot].double() * torch.mv(d["b"][slot].double(), torch.mv(d["a"][slot].double(), x[n]))
        return y
    tiles = y.reshape(N, M // 32, 32)
    g, u = tiles[:, :, :16].reshape(N, -1).clone().requires_grad_(), tiles[:, :, 16:].reshape(N, -1).clone().requires_grad_()
    del y, tiles
    F = torch.nn.functional
    if case["kind"] == "gated":
        with torch.no_grad():
            return (F.silu(g) if case["act"] == "silu" else F.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none")) * u
    h = (F.silu(g) if case["act"] == "silu" else F.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none")) * u
    dg, du = torch.autograd.grad(h, (g, u), d["dh"].double())
    dp = torch.empty(N, M // 32, 32, dtype=torch.float64, device=DEVICE)
    dp[:, :, :16], dp[:, :, 16:] = dg.reshape(N, -1, 16), du.reshape(N, -1, 16)
    dp = dp.reshape(N, M)
    dx = torch.zeros(N, K, dtype=torch.float64, device=DEVICE)
    for r in range(0, M, 4096):
        dx.addmm_(dp[:, r:r + 4096], W(r, r + 4096))
    return {"out": h.detach(), "grad_in": dx, "grad_preact": dp}
