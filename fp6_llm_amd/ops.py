"""Operators around the FPx linear layer, on the same native-layout weights: the gated feed-forward block with its backward pass, the input gradient of a
layer, and low-rank adapters of many requests beside a shared projection.  (The reference has the forward product alone.)

The functions enqueue on the current stream and check shapes, types and devices on the host, like linear_forward_native; what they compute is in include/fp6mi.h.  They go through
the torch extension where it is built (csrc/torch_binding.cpp makes the same checks), else through ctypes."""
import threading

import torch

from . import _lib

_HEURISTIC = -2 ** 63   # the extension's splitK for None
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
MAX_RANK = 256
_launch_lock = threading.Lock()   # the kernels of one call share a workspace: two threads on one stream must not interleave theirs (ctypes lets go of the interpreter's lock)


def gate_up_pairs(gate, up, rows=None):
    """Two equally shaped tensors about the same rows (weights [F, ...], scales or biases [F], or, with rows=F, native-layout weights or group exponents, whose
    16-row tiles lie one after another) as one tensor of 2F rows in pair order: 16 rows of gate, the same 16 of up, and so on."""
    F = gate.shape[0] if rows is None else rows
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise ValueError("gate and up must have the same shape, type and device")
    if F < 16 or F % 16 or gate.numel() % (F // 16):
        raise ValueError("pair order needs a multiple of 16 rows, got %d rows in %d elements" % (F, gate.numel()))
    pairs = torch.stack((gate.reshape(F // 16, -1), up.reshape(F // 16, -1)), 1)
    return pairs.reshape((2 * gate.shape[0],) + tuple(gate.shape[1:]))


def gradient_goes_elsewhere(t):
    """Whether a backward pass from t would reach a node that runs on another stream than the current one: of a graph that was made on that stream, a leaf's own node among them while
    such a graph lives.  (Without the extension, which can ask, nothing is known and the answer is True.)"""
    from . import _ext
    return _ext.gradient_goes_elsewhere(t) if _ext is not None else True


def _check_weights(E, M, native_weight, scales, OC, IC, group_exps, dev):
    from . import _BLOCK_BYTES, _bits, _check_group_exps
    bits = _bits(E, M)
    if OC < 256 or OC % 256 or IC < 64 or IC % 64:
        raise ValueError("need OC %% 256 == 0 and IC %% 64 == 0 (got OC=%d IC=%d)" % (OC, IC))
    if native_weight.device != dev or scales.device != dev:
        raise ValueError("activations, weights and scales must be on the same GPU")
    if not native_weight.is_contiguous() or native_weight.numel() * native_weight.element_size() != (OC // 16) * ((IC + 255) // 256) * _BLOCK_BYTES[bits]:
        raise ValueError("native_weight must be contiguous and of the size for OC=%d IC=%d" % (OC, IC))
    if scales.dtype != torch.float16 or scales.numel() != OC:
        raise ValueError("scales must be float16 [OC]")
    if group_exps is not None:
        _check_group_exps(group_exps, OC, IC, dev)


def _activations(t, name, cols=None):
    """t as contiguous float16 rows on a GPU."""
    if t.dtype != torch.float16 or t.dim() != 2 or t.device.type != "cuda":
        raise ValueError("%s must be a 2-D float16 tensor on the GPU" % name)
    if t.shape[0] < 1 or (cols is not None and t.shape[1] != cols):
        raise ValueError("%s must be [B >= 1, %s], got %s" % (name, "*" if cols is None else cols, list(t.shape)))
    return t.contiguous()


def _result(out, shape, dev, name="out", dtype=torch.float16):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if out.shape != shape or out.dtype != dtype or not out.is_contiguous() or out.device != dev:
        raise ValueError("%s must be a contiguous %s %s tensor on the same GPU" % (name, str(dtype).split(".")[-1], list(shape)))
    return out


def _vector(t, n, dtype, dev, name):
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
        raise ValueError("%s must be a contiguous %s [%d] tensor on the same GPU" % (name, str(dtype).split(".")[-1], n))
    return t


def _activation_code(activation):
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError("activation must be one of %s, got %r" % (", ".join(sorted(ACTIVATIONS)), activation)) from None


def _split(splitK, default):
    s = default() if splitK is None else int(splitK)
    if s < 1:
        raise ValueError("splitK must be >= 1")
    return s


def _launch(name, dev, need, workspace, call):
    """call(stream, workspace pointer) on the tensors' device and its current stream, with `need` bytes of scratch (beyond SPLIT_WORKSPACE_BYTES not kept for the next call)."""
    from . import SPLIT_WORKSPACE_BYTES, _workspace
    with torch.cuda.device(dev), _launch_lock:
        stream = torch.cuda.current_stream().cuda_stream
        if need and workspace is None:
            workspace = _workspace(dev, stream, need) if need <= SPLIT_WORKSPACE_BYTES else torch.empty((need + 3) // 4, dtype=torch.float32, device=dev)
        elif need and (workspace.dtype != torch.float32 or workspace.numel() * 4 < need or workspace.device != dev or not workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous float32 tensor of at least %d bytes on the same GPU" % need)
        _lib.check(call(stream, workspace.data_ptr() if need else None), name)


def _ptr(t):
    return None if t is None else t.data_ptr()


def gated_forward_native(EXPONENT, MANTISSA, in_feats, native_weight, scales, OC, activation="silu", splitK=None, out=None, preact=None, workspace=None, group_exps=None,
                         bias=None):
    """out[B, OC/2] = act(in_feats @ gate^T + bias_g) * (in_feats @ up^T + bias_u): both projections of a gated feed-forward block, the activation ("silu", "gelu",
    "gelu_tanh") and the product.  native_weight, scales, group_exps and bias are those of one matrix of OC = 2F rows in pair order (gate_up_pairs).
    preact: contiguous float32 [B, OC] that receives the pre-activations in pair order, for gated_backward_native.  splitK: None for the heuristic's."""
    from . import _ext, heuristic_splitk_mi355x
    act = _activation_code(activation)
    if _ext is not None:
        return _ext.gated_forward(EXPONENT, MANTISSA, in_feats, native_weight, scales, OC, act, _HEURISTIC if splitK is None else int(splitK), out, preact, workspace, group_exps, bias)
    x = _activations(in_feats, "in_feats")
    (B, IC), dev = x.shape, x.device
    _check_weights(EXPONENT, MANTISSA, native_weight, scales, OC, IC, group_exps, dev)
    s = _split(splitK, lambda: heuristic_splitk_mi355x(OC, B, IC, EXPONENT=EXPONENT, MANTISSA=MANTISSA))
    out = _result(out, (B, OC // 2), dev)
    if preact is not None:
        _result(preact, (B, OC), dev, "preact", torch.float32)
    if bias is not None:
        _vector(bias, OC, torch.float16, dev, "bias")
    sc, L = scales.contiguous(), _lib.lib()
    _launch("fp6mi_gated_native", dev, L.fp6mi_gated_workspace_bytes(OC, B, s), workspace, lambda stream, ws: L.fp6mi_gated_native(
        EXPONENT, MANTISSA, stream, native_weight.data_ptr(), sc.data_ptr(), _ptr(group_exps), _ptr(bias), x.data_ptr(), out.data_ptr(), _ptr(preact), OC, B, IC, act, ws, s))
    return out


def _grad_splits(E, M, OC, B, IC):
    from . import MI355X_CUS
    return _lib.lib().fp6mi_heuristic_grad_splits(E, M, OC, B, IC, MI355X_CUS)


def gated_backward_native(EXPONENT, MANTISSA, grad_out, preact, native_weight, scales, IC, activation="silu", splitK=None, grad_in=None, grad_preact=None, workspace=None,
                          group_exps=None):
    """The backward pass of gated_forward_native from grad_out [B, OC/2] and the preact [B, OC] it filled: (grad_in [B, IC], grad_preact [B, OC] in pair order).
    grad_preact is what a bias sums over the batch, or an adapter beside the block takes; False leaves it out (and None comes back).  The weights have no gradient."""
    from . import _ext
    act = _activation_code(activation)
    if _ext is not None:
        return _ext.gated_backward(EXPONENT, MANTISSA, grad_out, preact, native_weight, scales, IC, act, _HEURISTIC if splitK is None else int(splitK), grad_in,
                                   None if grad_preact is False else grad_preact, grad_preact is not False, workspace, group_exps)
    if preact.dtype != torch.float32 or preact.dim() != 2 or preact.device.type != "cuda" or not preact.is_contiguous():
        raise ValueError("preact must be the contiguous float32 [B, OC] tensor that gated_forward_native filled")
    (B, OC), dev = preact.shape, preact.device
    d = _activations(grad_out, "grad_out", OC // 2)
    if d.shape[0] != B or d.device != dev:
        raise ValueError("grad_out and preact must have the same rows, on the same GPU")
    _check_weights(EXPONENT, MANTISSA, native_weight, scales, OC, IC, group_exps, dev)
    s = _split(splitK, lambda: _grad_splits(EXPONENT, MANTISSA, OC, B, IC))
    grad_in = _result(grad_in, (B, IC), dev, "grad_in")
    grad_preact = None if grad_preact is False else _result(grad_preact, (B, OC), dev, "grad_preact")
    sc, L = scales.contiguous(), _lib.lib()
    _launch("fp6mi_gated_backward_native", dev, L.fp6mi_gated_backward_workspace_bytes(OC, B, IC, s), workspace, lambda stream, ws: L.fp6mi_gated_backward_native(
        EXPONENT, MANTISSA, stream, native_weight.data_ptr(), sc.data_ptr(), _ptr(group_exps), d.data_ptr(), preact.data_ptr(), _ptr(grad_preact), grad_in.data_ptr(),
        OC, B, IC, act, ws, s))
    return grad_in, grad_preact


def linear_input_grad_native(EXPONENT, MANTISSA, grad_out, native_weight, scales, IC, splitK=None, out=None, workspace=None, group_exps=None):
    """out[B, IC] = grad_out[B, OC] @ dequant(W): the gradient of linear_forward_native with respect to in_feats, from the same native-layout weights.
    (grad_out times the mantissa of a row's scale is rounded to float16 once, the products are summed in float32.)  splitK: parts of the sum over OC, None for the heuristic's."""
    from . import _ext
    if _ext is not None:
        return _ext.linear_input_grad(EXPONENT, MANTISSA, grad_out, native_weight, scales, IC, _HEURISTIC if splitK is None else int(splitK), out, workspace, group_exps)
    d = _activations(grad_out, "grad_out")
    (B, OC), dev = d.shape, d.device
    _check_weights(EXPONENT, MANTISSA, native_weight, scales, OC, IC, group_exps, dev)
    s = _split(splitK, lambda: _grad_splits(EXPONENT, MANTISSA, OC, B, IC))
    out = _result(out, (B, IC), dev)
    sc, L = scales.contiguous(), _lib.lib()
    _launch("fp6mi_linear_grad_native", dev, L.fp6mi_grad_workspace_bytes(B, IC, s), workspace, lambda stream, ws: L.fp6mi_linear_grad_native(
        EXPONENT, MANTISSA, stream, native_weight.data_ptr(), sc.data_ptr(), _ptr(group_exps), d.data_ptr(), out.data_ptr(), OC, B, IC, ws, s))
    return out


def adapter_forward_native(EXPONENT, MANTISSA, in_feats, native_weight, scales, OC, lora_a, lora_b, scaling, index, splitK=None, out=None, workspace=None, group_exps=None,
                           bias=None):
    """linear_forward_native with a low-rank adapter for every row of the batch:
    out[n] = in_feats[n] @ dequant(W)^T + bias + scaling[a] * (in_feats[n] @ lora_a[a]^T) @ lora_b[a]^T,  a = index[n].
    lora_a: float16 [slots, R, IC], lora_b: float16 [slots, OC, R], scaling: float32 [slots], index: int32 [B], all on the GPU; a row whose index is no slot's number (-1,
    say) has no adapter.  R is a multiple of 8 up to 256: pad smaller ranks with zeros.  The layer's output is rounded to float16 before the adapter's part is added to it, which is
    rounded once more; of that part the rank sums in_feats[n] @ lora_a[a]^T are held to 2^-11 of themselves in large batches, to 2^-22 in small ones."""
    from . import _ext, heuristic_splitk_mi355x
    if _ext is not None:
        return _ext.adapter_forward(EXPONENT, MANTISSA, in_feats, native_weight, scales, OC, lora_a, lora_b, scaling, index, _HEURISTIC if splitK is None else int(splitK), out,
                                    workspace, group_exps, bias)
    x = _activations(in_feats, "in_feats")
    (B, IC), dev = x.shape, x.device
    _check_weights(EXPONENT, MANTISSA, native_weight, scales, OC, IC, group_exps, dev)
    if lora_a.dim() != 3 or lora_a.shape[2] != IC or lora_a.shape[0] < 1:
        raise ValueError("lora_a must be [slots, R, IC=%d], got %s" % (IC, list(lora_a.shape)))
    slots, R = lora_a.shape[:2]
    if R < 8 or R % 8 or R > MAX_RANK:
        raise ValueError("the rank must be a multiple of 8 up to %d, got %d" % (MAX_RANK, R))
    if lora_b.shape != (slots, OC, R):
        raise ValueError("lora_b must be [slots=%d, OC=%d, R=%d], got %s" % (slots, OC, R, list(lora_b.shape)))
    for t, name in ((lora_a, "lora_a"), (lora_b, "lora_b")):
        if t.dtype != torch.float16 or not t.is_contiguous() or t.device != dev:
            raise ValueError("%s must be contiguous float16 on the same GPU" % name)
    _vector(scaling, slots, torch.float32, dev, "scaling")
    _vector(index, B, torch.int32, dev, "index")
    if bias is not None:
        _vector(bias, OC, torch.float16, dev, "bias")
    s = _split(splitK, lambda: heuristic_splitk_mi355x(OC, B, IC, EXPONENT=EXPONENT, MANTISSA=MANTISSA))
    out = _result(out, (B, OC), dev)
    sc, L = scales.contiguous(), _lib.lib()
    _launch("fp6mi_adapter_native", dev, L.fp6mi_adapter_workspace_bytes(OC, B, IC, R, s), workspace, lambda stream, ws: L.fp6mi_adapter_native(
        EXPONENT, MANTISSA, stream, native_weight.data_ptr(), sc.data_ptr(), _ptr(group_exps), _ptr(bias), x.data_ptr(), out.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(),
        scaling.data_ptr(), index.data_ptr(), OC, B, IC, R, slots, ws, s))
    return out
