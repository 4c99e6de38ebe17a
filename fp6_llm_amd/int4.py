"""Products with 4-bit integer weights that carry a scale, and possibly a zero point, for each row and group of columns: w[m,k] = s[m,g] * (q[m,k] - z[m,g]).  (The reference has FPx weights with
one scale a row.)  Activations and scales are float16 or bfloat16; products are exact, sums float32, rounded once.

The functions enqueue on the current stream and check shapes, types and devices on the host, like linear_forward_native; what they compute is in include/fp6mi.h.  They go through the torch extension
where it is built, else through ctypes."""
import sys

import torch

from . import _lib, ops

_package = sys.modules[__package__]   # (an attribute of it takes a tenth of the time of an import in a call)

TYPES = {torch.float16: 0, torch.bfloat16: 1}


def int4_quantize(weight, group=128, zeros=False):
    """codes uint8 [..., OC, IC/2], scales [..., OC, ceil(IC/group)] and zero points (uint8 like the scales, or None) of a float16, bfloat16 or float32 weight [..., OC, IC], rounded to nearest.
    Without zero points the codes are 1..15 about 8 and a scale is the group's largest magnitude / 7; with them a group's range (0 included) is cut into 15 steps.
    Scales have the weight's type, float16 for float32; a weight that they do not reach, or that is not finite, is refused (which waits for a GPU)."""
    if weight.dtype not in (torch.float16, torch.bfloat16, torch.float32) or weight.dim() < 2 or weight.shape[-1] % 2 or weight.numel() == 0:
        raise ValueError("weight must be float16, bfloat16 or float32 [..., OC, IC], IC even")
    if group < 32 or group % 32:
        raise ValueError("group must be a positive multiple of 32, got %d" % group)
    dtype = torch.float16 if weight.dtype == torch.float32 else weight.dtype
    IC = weight.shape[-1]
    groups = (IC + group - 1) // group
    w = torch.nn.functional.pad(weight.detach().float(), (0, groups * group - IC)).unflatten(-1, (groups, group))   # (zeros in a cut group change neither its range nor its largest magnitude)
    if not zeros:
        scales, z = (w.abs().amax(-1) / 7).to(dtype), None
    else:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((high - low) / 15).to(dtype)
        z = torch.where(scales > 0, torch.round(-low / scales.float()), 0).clamp(0, 15)
    if not bool(scales.isfinite().all()):
        raise ValueError("the weight holds infinities, NaN or values beyond what scales in %s reach" % str(dtype).split(".")[-1])
    step = torch.where(scales > 0, scales.float(), 1.0).unsqueeze(-1)
    q = torch.round(w / step).add_(8 if z is None else z.unsqueeze(-1)).clamp_(0 if zeros else 1, 15).to(torch.uint8).flatten(-2)[..., :IC]
    return q[..., 0::2] | q[..., 1::2] << 4, scales, None if z is None else z.to(torch.uint8)


def native_shapes(OC, IC, group, zeros, experts=None):
    """Of the native weights (int32) and scales of int4_pack_native."""
    lead = (() if experts is None else (experts,)) + (OC // 16, (IC + 127) // 128)
    return lead + (256,), lead + (16, 128 // (128 if group % 128 == 0 else 64 if group % 64 == 0 else 32), 2 if zeros else 1)


def int4_pack_native(codes, scales, zeros=None, group=128):
    """(native_weight, native_scales) of int4_forward_native from weights as a checkpoint holds them: codes uint8 [OC, IC/2], two to a byte, the even column in the low half; scales float16 or
    bfloat16 [OC, ceil(IC/group)]; zeros uint8 like the scales, 0..15, or None: 8 everywhere.  Or all three for experts, [E, ...].  On the tensors' device, a GPU's or the host's.
    The native scales' shape holds the rest: [(E,) OC/16, ceil(IC/128), 16, 128/group, 2 with zero points else 1], where a group is the largest of 128, 64 and 32 columns that divides `group`."""
    if codes.dtype != torch.uint8 or codes.dim() not in (2, 3):
        raise ValueError("codes must be uint8 [OC, IC/2] or [E, OC, IC/2]")
    OC, IC = codes.shape[-2], 2 * codes.shape[-1]
    E = codes.shape[0] if codes.dim() == 3 else 1
    if OC < 16 or OC % 16 or IC < 32 or IC % 32 or E < 1:
        raise ValueError("need OC %% 16 == 0 and IC %% 32 == 0 (got OC=%d IC=%d)" % (OC, IC))
    if group < 32 or group % 32:
        raise ValueError("group must be a positive multiple of 32, got %d" % group)
    shape = codes.shape[:-1] + ((IC + group - 1) // group,)
    if scales.dtype not in TYPES or scales.shape != shape or scales.device != codes.device:
        raise ValueError("scales must be float16 or bfloat16 %s on the codes' device, got %s %s" % (list(shape), str(scales.dtype).split(".")[-1], list(scales.shape)))
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != shape or zeros.device != codes.device):
        raise ValueError("zeros must be uint8 %s on the codes' device" % list(shape))
    if codes.device.type not in ("cuda", "cpu"):
        raise ValueError("codes must be on a GPU or on the host")
    native, native_scales = native_shapes(OC, IC, group, zeros is not None, E if codes.dim() == 3 else None)
    w, s = torch.empty(native, dtype=torch.int32, device=codes.device), torch.empty(native_scales, dtype=scales.dtype, device=codes.device)
    codes, scales, zeros = codes.contiguous(), scales.resolve_neg().contiguous(), None if zeros is None else zeros.contiguous()
    args = (w.data_ptr(), s.data_ptr(), codes.data_ptr(), scales.data_ptr(), ops._ptr(zeros), TYPES[scales.dtype], E, OC, IC, group)
    if codes.device.type == "cpu":
        _lib.check(_lib.lib().fp6mi_int4_pack(*args), "fp6mi_int4_pack")
    else:
        with torch.cuda.device(codes.device):
            _lib.check(_lib.lib().fp6mi_int4_pack_gpu(torch.cuda.current_stream().cuda_stream, *args), "fp6mi_int4_pack_gpu")
    return w, s


def _overlap(a, b):
    return a.data_ptr() < b.data_ptr() + b.numel() * b.element_size() and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


def int4_forward_native(in_feats, native_weight, native_scales, plan=None, activation=None, bias=None, out=None, out_dtype=None, workspace=None):
    """out[B, OC] = in_feats[B, IC] @ w^T (+ bias[OC]) with the weights of int4_pack_native.  activation ("silu", "gelu", "gelu_tanh"): out[B, OC/2] = act(gate) * up, for weights (and bias) whose
    rows are in pair order (16 rows of gate, the same 16 of up, and so on: gate_up_pairs).
    plan: that of expert_sort or expert_plan, for the weights of experts [E, ...] (bias [E, OC]): rows sorted by expert, each multiplied with its expert's weights; rows behind those come out as zeros.
    IC is that of the weights, which their native shape tells to 128 columns only.  in_feats has the scales' type, out too or (out_dtype) float32; out may not lie over an input.  workspace: float32, of fp6mi_int4_workspace_bytes (many bfloat16 rows need one).  The product has no gradient: inputs that are to get one, tangents, transforms of torch.func and traces are refused."""
    _ext = _package._ext
    act = -1 if activation is None else ops._activation_code(activation)
    f32 = out_dtype == torch.float32
    if out_dtype is not None and not f32 and out_dtype != native_scales.dtype:
        raise ValueError("out_dtype must be float32 or the scales' type")
    if _ext is not None:
        if plan is None:
            return _ext.int4_forward(in_feats, native_weight, native_scales, None, 0, 0, act, bias, out, f32, workspace)
        return _ext.int4_forward(in_feats, native_weight, native_scales, plan.table, plan.experts, plan.places, act, bias, out, f32, workspace)
    seen = [t for t in (in_feats, native_scales, bias) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in seen):
        raise ValueError("a product with 4-bit weights has no gradient: call it under torch.no_grad()")
    _refuse_unseen(*seen)
    s, bias = native_scales.resolve_neg(), None if bias is None else bias.resolve_neg()
    dims = 6 if plan is not None else 5
    if s.dtype not in TYPES or s.dim() != dims or s.shape[-3] != 16 or s.shape[-2] not in (1, 2, 4) or s.shape[-1] not in (1, 2) or not s.is_contiguous():
        raise ValueError("native_scales must be those of int4_pack_native, %s" % ("of experts" if plan is not None else "of one matrix"))
    x, dev = in_feats, s.device
    if x.dtype != s.dtype or x.dim() != 2 or x.device.type != "cuda" or x.device != dev or native_weight.device != dev:
        raise ValueError("in_feats must be 2-D of the scales' type, on the weights' GPU")
    B, IC = x.shape
    tiles, KB = s.shape[-5], s.shape[-4]
    OC = 16 * tiles
    if IC < 32 or IC % 32 or (IC + 127) // 128 != KB:
        raise ValueError("in_feats has IC=%d columns, the weights have %d blocks of 128" % (IC, KB))
    if native_weight.dtype != torch.int32 or native_weight.shape != s.shape[:-3] + (256,) or not native_weight.is_contiguous():
        raise ValueError("native_weight must be that of int4_pack_native with these scales")
    if act >= 0 and OC % 32:
        raise ValueError("a gated product needs OC %% 32 == 0, got %d" % OC)
    E, offsets = 1, None
    if plan is not None:
        E = s.shape[0]
        if plan.experts != E or plan.table.device != dev or B != plan.places:
            raise ValueError("the plan must be of %d experts and as many places as in_feats has rows, on the same GPU" % E)
        offsets = plan._addresses()[0]
    if bias is not None and (bias.dtype != s.dtype or bias.shape != ((E, OC) if plan is not None else (OC,)) or not bias.is_contiguous() or bias.device != dev):
        raise ValueError("bias must be contiguous, of the scales' type, one for each row of the weights, on the same GPU")
    x = x.resolve_neg().contiguous()
    if out is not None and (out.is_neg() or any(_overlap(out, t) for t in (x, native_weight, s, bias) if t is not None)):
        raise ValueError("out must have memory of its own, and be no negative view")
    out = ops._result(out, (B, OC // 2 if act >= 0 else OC), dev, dtype=torch.float32 if f32 else s.dtype)
    L = _lib.lib()
    ops._launch("fp6mi_int4_linear", dev, L.fp6mi_int4_workspace_bytes(TYPES[s.dtype], 128 // s.shape[-2], E, plan is not None, OC, B, IC, act >= 0, -1), workspace, lambda stream, ws: L.fp6mi_int4_linear(
        stream, TYPES[s.dtype], native_weight.data_ptr(), s.data_ptr(), 128 // s.shape[-2], s.shape[-1] - 1, ops._ptr(bias), x.data_ptr(), out.data_ptr(), f32, act, offsets, E, OC, B, IC, ws))
    return out


from .module import _refuse_unseen  # noqa: E402  (it imports this module)
