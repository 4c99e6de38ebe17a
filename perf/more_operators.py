"""Timed cases of the operators for 4-bit integer weights with a scale for each group of columns, and for mixtures of experts: the product with such weights (one matrix, or the
gated projections of many experts with rows sorted by expert), tokens sorted by expert, and the experts' rows weighted and summed back to tokens, each with its gradient.

`own` chooses between the package's entry points and a plain form in elementary torch operations, 32 bits throughout.  Weights are given as a checkpoint holds them: two codes of
4 bits to a byte (the even column in the low half), a scale and, with zeros, a zero point of 4 bits for each row and group; the package's side holds them in its native layout, as a program
that has loaded a checkpoint does.  M = weight rows, K = input features, N = tokens, F = outputs of a gated projection, H = row length, k = experts of a token, E = experts.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MAX_FLOPS = 2 * 2048 * 2 * 22016 * 4096   # the largest listed case
MAX_BYTES = 1 << 30


def _int4(name, M, K, N, group=128, zeros=False, type="fp16", bias=False):
    return {"name": name, "kind": "int4", "M": M, "K": K, "N": N, "group": group, "zeros": zeros, "type": type, "bias": bias}


def _experts(name, F, K, N, k, E, group=128, zeros=False, type="fp16", drop=0.0, act="silu"):
    return {"name": name, "kind": "experts", "F": F, "K": K, "N": N, "k": k, "E": E, "group": group, "zeros": zeros, "type": type, "drop": drop, "act": act}


def _rows(kind, name, H, N, k, E, type="fp16", drop=0.0, train=False):
    return {"name": name, "kind": kind, "H": H, "N": N, "k": k, "E": E, "type": type, "drop": drop, "train": train}


def listed():
    return [
        # one token through a projection of a small model: the call's own latency counts
        _int4("int4_4096x4096_n1", 4096, 4096, 1),
        # four requests on a large matrix with zero points, in bfloat16
        _int4("int4_28672x8192_n4_bf16_zeros", 28672, 8192, 4, 64, True, "bf16"),
        # an odd batch, the finest groups, columns that end inside a block, a bias
        _int4("int4_10240x4576_n19_g32_zeros", 10240, 4576, 19, 32, True, "fp16", True),
        # a short prompt of odd length
        _int4("int4_8192x8192_n777", 8192, 8192, 777),
        # one token of a model with a few large experts: two of eight are read
        _experts("experts_11008x4096_n1_2of8", 11008, 4096, 1, 2, 8),
        # a decode batch over many small experts: a few rows to each
        _experts("experts_1280x2048_n40_8of64", 1280, 2048, 40, 8, 64, 64, True, "bf16"),
        # a prompt chunk over large experts: the largest case
        _experts("experts_11008x4096_n2048_2of8", 11008, 4096, 2048, 2, 8),
        # a decode batch sorted by expert; a training batch of odd length with padded tokens (no expert), rows and the gradient of the tokens
        _rows("sort", "sort_4096_n16_4of64", 4096, 16, 4, 64),
        _rows("sort", "sort_train_4096_n4099_2of8", 4096, 4099, 2, 8, "bf16", 0.05, True),
        # a token's eight experts summed; training batches: the sum, the gradients of the rows and of the weights (the second with rows of odd length, which no vector load fits)
        _rows("combine", "combine_8192_n1_8of64", 8192, 1, 8, 64),
        _rows("combine", "combine_train_4096_n8192_4of64", 4096, 8192, 4, 64, "bf16", 0.0, True),
        _rows("combine", "combine_train_2305_n333_3of5", 2305, 333, 3, 5, "fp32", 0.1, True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("int4", "experts", "sort", "combine"))
    E = log(2, 128)
    k, drop = rng.randint(1, min(8, E)), rng.choice((0.0, 0.0, 0.1))
    group, zeros, type = rng.choice((32, 64, 128)), rng.random() < 0.5, rng.choice(("fp16", "bf16"))
    while True:
        if kind == "int4":
            case = _int4("", 16 * log(16, 1792), 32 * log(16, 256), log(1, 1024), group, zeros, type, rng.random() < 0.3)
            fits = 2 * case["N"] * case["M"] * case["K"] <= MAX_FLOPS // 2
        elif kind == "experts":
            case = _experts("", 16 * log(16, 688), 32 * log(16, 128), log(1, 2048), k, E, group, zeros, type, drop, rng.choice(("silu", "gelu", "gelu_tanh")))
            fits = 4 * case["N"] * k * case["F"] * case["K"] <= MAX_FLOPS // 2 and case["F"] * case["K"] * E <= MAX_BYTES // 2
        else:
            case = _rows(kind, "", log(128, 8192), log(1, 8192), k, E, rng.choice(("fp16", "bf16", "fp32")), drop, rng.random() < 0.5)
            fits = 4 * case["N"] * k * case["H"] <= MAX_BYTES // 2
        if fits:
            del case["name"]
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _weights(g, case, E, M):
    """codes uint8 [E, M, K/2], scales [E, M, groups] and zero points uint8 like them (None: 8 everywhere) of weights of about normal values, quantized by groups of columns."""
    K, groups = case["K"], (case["K"] + case["group"] - 1) // case["group"]
    codes = torch.empty(E, M, K // 2, device=DEVICE, dtype=torch.uint8)
    for e in range(E):   # a sum of three dice is bell-shaped over the codes
        low, high = (sum(torch.randint(0, 6, (M, K // 2), generator=g, device=DEVICE, dtype=torch.uint8) for _ in range(3)) for _ in range(2))
        codes[e] = low + 16 * high
    spread = torch.exp(0.3 * torch.randn(E, M, groups, generator=g, device=DEVICE))
    scales = (spread / (3.0 * math.sqrt(K))).to(TYPES[case["type"]])
    zeros = torch.randint(5, 11, (E, M, groups), generator=g, device=DEVICE, dtype=torch.uint8) if case["zeros"] else None
    return codes, scales, zeros


def _router(g, case):
    """index int64 [N, k]: the experts of every token, some of them busier than others, no expert twice; -1 for a share of the places.  weights float32 [N, k]: their softmax."""
    N, k, E = case["N"], case["k"], case["E"]
    logits = torch.randn(N, E, generator=g, device=DEVICE) + 0.5 * torch.randn(E, generator=g, device=DEVICE)
    top = logits.topk(k, 1)
    weights = torch.exp(top.values - top.values[:, :1])
    weights = weights / weights.sum(1, keepdim=True)
    index = top.indices
    if case["drop"]:
        index = torch.where(torch.rand(N, k, generator=g, device=DEVICE) < case["drop"], torch.full_like(index, -1), index)
    return index, weights


def _order(index, E):
    """Places of index in order of their experts (ties in their own order, those without an expert last), and how many each expert has."""
    keys = index.reshape(-1)
    keys = torch.where((keys < 0) | (keys >= E), torch.full_like(keys, E), keys)
    order = torch.sort(keys, stable=True).indices
    return order, (keys.unsqueeze(0) == torch.arange(E, device=DEVICE).unsqueeze(1)).sum(1)


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    type, kind = TYPES[case["type"]], case["kind"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)   # noqa: E731
    d = {}
    if kind == "int4":
        d["codes"], d["scales"], d["zeros"] = (t if t is None else t[0] for t in _weights(g, case, 1, case["M"]))
        d["x"] = randn(case["N"], case["K"]).to(type)
        d["bias"] = (0.1 * randn(case["M"])).to(type) if case["bias"] else None
        return d
    d["index"], d["weights"] = _router(g, case)
    if kind == "experts":
        d["codes"], d["scales"], d["zeros"] = _weights(g, case, case["E"], 2 * case["F"])
        d["x"] = randn(case["N"], case["K"]).to(type)
    elif kind == "sort":
        d["x"] = randn(case["N"], case["H"]).to(type)
        d["grad"] = (0.1 * randn(case["N"] * case["k"], case["H"])).to(type) if case["train"] else None
    else:
        d["rows"] = randn(case["N"] * case["k"], case["H"]).to(type)
        d["grad"] = (0.1 * randn(case["N"], case["H"])).to(type) if case["train"] else None
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    state = {"case": case, **d}
    if own:
        import fp6_llm_amd as fp6
        if "codes" in d:
            state["w"], state["sc"] = fp6.int4_pack_native(d["codes"], d["scales"], d["zeros"], case["group"])
            del state["codes"], state["scales"], state["zeros"]
    if kind == "experts":   # the rows as the sort in front of the product leaves them, and its plan
        if own:
            state["x"], state["plan"] = fp6.expert_sort(d["x"], d["index"], case["E"])
        else:
            order, counts = _order(d["index"], case["E"])
            state["x"], state["counts"] = d["x"][order // case["k"]], counts.tolist()
    elif kind == "combine":
        if own:   # (a plan is made of an index; its rows here come from a model's experts)
            state["plan"] = fp6.expert_plan(d["index"], case["E"])
        else:
            order, counts = _order(d["index"], case["E"])
            state["place"], state["valid"] = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=DEVICE)), int(counts.sum())
    if kind in ("sort", "combine") and case["train"]:
        for name in ("x", "rows", "weights"):
            if name in state and (kind == "combine" or name == "x"):
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def _act(act, g):
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def _halves(p):
    """Pair order (16 gate rows, the same 16 of up, ...) -> gate and up."""
    p = p.view(p.shape[0], -1, 2, 16)
    return p[:, :, 0].flatten(1), p[:, :, 1].flatten(1)


def _dequantized(codes, scales, zeros, group):
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    each = torch.arange(q.shape[-1], device=DEVICE) // group
    q -= 8.0 if zeros is None else zeros.float()[..., each]
    return q.mul_(scales.float()[..., each])


@torch.no_grad()
def _plain(s):
    c = s["case"]
    type, kind = TYPES[c["type"]], c["kind"]
    if kind == "int4":
        y = s["x"].float() @ _dequantized(s["codes"], s["scales"], s["zeros"], c["group"]).t()
        return (y if s["bias"] is None else y + s["bias"].float()).to(type)
    if kind == "experts":
        x, at = s["x"].float(), 0
        out = torch.zeros(x.shape[0], c["F"], device=DEVICE)
        for e, n in enumerate(s["counts"]):
            if n:
                g, u = _halves(x[at:at + n] @ _dequantized(s["codes"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e], c["group"]).t())
                out[at:at + n] = _act(c["act"], g) * u
            at += n
        return out.to(type)
    k = c["k"]
    if kind == "sort":
        order, counts = _order(s["index"], c["E"])
        valid = torch.arange(order.numel(), device=DEVICE) < counts.sum()
        out = {"rows": torch.where(valid[:, None], s["x"][order // k], 0), "order": torch.where(valid, order, -1).int(), "offsets": torch.cat((torch.zeros_like(counts[:1]), counts.cumsum(0))).int()}
        if c["train"]:
            g = torch.where(valid[:, None], s["grad"].float(), 0)
            place = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=DEVICE))
            out["grad_x"] = g[place].view(c["N"], k, -1).sum(1).to(type)
        return out
    valid = (s["place"] < s["valid"]).view(-1, k, 1)
    rows = s["rows"].float()[s["place"]].view(c["N"], k, -1)
    out = {"out": torch.where(valid, s["weights"][:, :, None] * rows, 0).sum(1).to(type)}
    if c["train"]:
        g = s["grad"].float()[:, None]
        out["grad_weights"] = torch.where(valid, g * rows, 0).sum(2)
        grad_rows = torch.where(valid, s["weights"][:, :, None] * g, 0).flatten(0, 1)
        out["grad_rows"] = torch.empty_like(s["rows"]).index_copy_(0, s["place"], grad_rows.to(type))
    return out


def _own(s):
    import fp6_llm_amd as fp6
    c = s["case"]
    kind = c["kind"]
    if kind == "int4":
        return fp6.int4_forward_native(s["x"], s["w"], s["sc"], bias=s["bias"])
    if kind == "experts":
        return fp6.int4_forward_native(s["x"], s["w"], s["sc"], plan=s["plan"], activation=c["act"])
    if kind == "sort":
        rows, plan = fp6.expert_sort(s["x"], s["index"], c["E"])
        out = {"rows": rows, "order": plan.order, "offsets": plan.offsets}
        if c["train"]:
            out["grad_x"], = torch.autograd.grad(rows, s["x"], s["grad"])
        return out
    y = fp6.expert_combine(s["rows"], s["plan"], s["weights"])
    if not c["train"]:
        return {"out": y}
    grad_rows, grad_weights = torch.autograd.grad(y, (s["rows"], s["weights"]), s["grad"])
    return {"out": y, "grad_weights": grad_weights, "grad_rows": grad_rows}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------- what a pass is measured against
def work(case):
    size, N = (4 if case["type"] == "fp32" else 2), case["N"]
    if case["kind"] in ("int4", "experts"):
        K, groups = case["K"], (case["K"] + case["group"] - 1) // case["group"]
        M = case["M"] if case["kind"] == "int4" else 2 * case["F"]
        weights = M * K // 2 + M * groups * (2.5 if case["zeros"] else 2)
        if case["kind"] == "int4":
            return {"bytes": weights + 2 * N * (K + M) + (2 * M if case["bias"] else 0), "flops": 2 * N * M * K}
        pairs = N * case["k"] * (1 - case["drop"])   # (each expert's weights are read where it has a row: of N choices of k experts of E)
        used = case["E"] * (1 - (1 - case["k"] * (1 - case["drop"]) / case["E"]) ** N)
        return {"bytes": used * weights + 2 * pairs * (K + case["F"]), "flops": 2 * pairs * M * K}
    H, pairs = case["H"], N * case["k"]
    if case["kind"] == "sort":   # tokens and index in, rows, order and offsets out; the rows' gradient in, the tokens' out
        step = size * H * (N + pairs)
        return {"bytes": step * (2 if case["train"] else 1) + 12 * pairs + 4 * case["E"], "flops": pairs * H if case["train"] else 0}
    step = size * H * (N + pairs)   # rows in, tokens out; the tokens' gradient and rows in, the rows' gradient out
    return {"bytes": step + (size * H * (N + 2 * pairs) + 4 * pairs if case["train"] else 0) + 8 * pairs, "flops": pairs * H * (5 if case["train"] else 2)}


@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits, a slice of weight rows or a place of the tokens' experts at a time."""
    d = _inputs(case, seed)
    kind = case["kind"]

    def weight(e, lo, hi):
        codes, scales, zeros = (t if t is None or kind == "int4" else t[e] for t in (d["codes"], d["scales"], d["zeros"]))
        w = torch.empty(hi - lo, case["K"], dtype=torch.float64, device=DEVICE)
        w[:, 0::2], w[:, 1::2] = codes[lo:hi].remainder(16), codes[lo:hi].div(16, rounding_mode="floor")
        for j in range(scales.shape[1]):
            part = w[:, j * case["group"]:(j + 1) * case["group"]]
            part.sub_(8 if zeros is None else zeros[lo:hi, j:j + 1].double()).mul_(scales[lo:hi, j:j + 1].double())
        return w

    if kind == "int4":
        M = case["M"]
        y = torch.cat([torch.mm(d["x"].double(), weight(0, r, min(M, r + 4096)).t()) for r in range(0, M, 4096)], 1)
        return y if d["bias"] is None else y.add_(d["bias"].double())
    N, k, E = case["N"], case["k"], case["E"]
    experts = d["index"].flatten().tolist()
    sorted_places = [p for e in range(E) for p in range(N * k) if experts[p] == e] if N * k * E <= 1 << 16 else sorted((p for p in range(N * k) if 0 <= experts[p] < E), key=lambda p: experts[p])
    n = len(sorted_places)
    places = torch.tensor(sorted_places, dtype=torch.int64, device=DEVICE)
    if kind == "experts":
        F = torch.nn.functional
        out = torch.zeros(N * k, case["F"], dtype=torch.float64, device=DEVICE)
        at = 0
        for e in range(E):
            mine = experts.count(e)
            if mine:
                x = d["x"][places[at:at + mine] // k].double()
                for r in range(0, 2 * case["F"], 4096):
                    hi = min(2 * case["F"], r + 4096)
                    tiles = torch.mm(x, weight(e, r, hi).t()).reshape(mine, (hi - r) // 32, 32)
                    g, u = tiles[:, :, :16].reshape(mine, -1), tiles[:, :, 16:].reshape(mine, -1)
                    a = F.silu(g) if case["act"] == "silu" else F.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
                    out[at:at + mine, r // 2:hi // 2] = a * u
            at += mine
        return out
    H = case["H"]
    if kind == "sort":
        rows = torch.zeros(N * k, H, dtype=torch.float64, device=DEVICE)
        rows[:n] = d["x"].double()[places // k]
        out = {"rows": rows, "order": None, "offsets": None}
        if case["train"]:
            out["grad_x"] = torch.zeros(N, H, dtype=torch.float64, device=DEVICE).index_add_(0, places // k, d["grad"][:n].double())
        return out
    out = {"out": torch.zeros(N, H, dtype=torch.float64, device=DEVICE)}
    if case["train"]:
        out["grad_weights"] = torch.zeros(N, k, dtype=torch.float64, device=DEVICE)
        out["grad_rows"] = torch.zeros(N * k, H, dtype=torch.float64, device=DEVICE)
    for j in range(k):
        mine = (places % k == j).nonzero()[:, 0]
        tokens, w = places[mine] // k, d["weights"][:, j].double()
        row = d["rows"][mine].double()
        out["out"][tokens] += w[tokens, None] * row
        if case["train"]:
            g = d["grad"][tokens].double()
            out["grad_weights"][tokens, j] = (g * row).sum(1)
            out["grad_rows"][mine] = w[tokens, None] * g
    return out
