"""Caller-side conveniences around the linear-layer path: a torch module that owns native-layout weights, and a small
on-disk container for them.  (The reference leaves both to the framework that embeds it -- DeepSpeed, README.md:19.)"""
import json
import struct
import sys

import numpy as np
import torch

from . import quant
from . import (MI355X_CUS, group_exps_bytes, heuristic_splitk_mi355x, linear_forward_native, native_bytes, pack_group_exps, to_native,
               weight_dequant_native_cuda, weight_prepacking_native_cpu, weight_quantize_native_cuda)
from . import ops

_MAGIC = b"FP6MI\x00\x01\x00"   # name, NUL, layout version 1, reserved


_peek_transform = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", None)
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_forward_ad, _is_compiling, _is_tracing = torch.autograd.forward_ad, torch.compiler.is_compiling, torch.jit.is_tracing


def _values_only(t):
    """Whether nothing but t's values counts in what is done with it: no derivative, transform, trace, subclass or dispatch mode has a part in it, which a kernel
    that is handed t's address would pass by.  (A torch that lacks one of the names asked here is taken to have one of these active.)"""
    return (type(t) in (torch.Tensor, torch.nn.Parameter) and not (t.requires_grad and torch.is_grad_enabled())
            and _peek_transform is not None and _peek_transform() is None and getattr(torch.autograd.forward_ad, "_current_level", 0) < 0
            and _dispatch_modes is not None and _dispatch_modes() == 0 and not torch.jit.is_tracing() and not t.is_neg())


class _AutoRows(int):
    """What dequant_above reads under "auto": the number of rows, and "auto" again for a module that it is assigned to.  (Modules that library version 139
    pickled whole hold one.)"""


def _differentiates(x):
    """Whether a gradient is to reach x.  A backward pass that is captured must stay on its stream: where x, or a leaf that it was computed from, is also part of an eager graph that
    still lives, its gradient is added up on that graph's stream, and a capture that goes there ends the process.  A call that would begin one is refused."""
    if not (x.requires_grad and torch.is_grad_enabled()):
        return False
    if x.device.type == "cuda" and torch.cuda.is_current_stream_capturing() and ops.gradient_goes_elsewhere(x):
        raise RuntimeError("the gradient of this input would leave the stream that is being captured: drop what an eager graph holds of it, or capture a detached copy that requires it")
    return True


def _refuse_unseen(x):
    """What a kernel that is handed x's address would pass by in silence: a tangent that x carries (forward mode), a transform of torch.func that x is part of, a trace that is being made,
    which would record the output as it was allocated and not what fills it."""
    if _is_compiling():   # (a call of a kernel ends the graph that is compiled)
        return
    wrapped = _peek_transform is None or (_peek_transform() is not None and torch._C._functorch.is_functorch_wrapped_tensor(x))
    if wrapped or (getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(x).tangent is not None):
        raise RuntimeError("this operator has no part in forward mode or in a transform of torch.func")
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")   # (not loaded: no such trace is being made)
    if _is_tracing() or (proxies is not None and proxies.get_proxy_mode() is not None):
        raise RuntimeError("this operator cannot be recorded by a trace")


def _held(module, name):
    """A buffer of a module, which as an attribute takes half a microsecond; or whatever has taken its place."""
    held = module._buffers
    return held[name] if name in held else getattr(module, name)


def _rows_of(x, features):
    """x[..., features] as float16 rows, of which nothing but their values counts or a backward pass."""
    _refuse_unseen(x)
    if x.dim() < 1 or x.shape[-1] != features:
        raise ValueError("need an input of %d features, got %s" % (features, list(x.shape)))
    x2 = x.reshape(-1, features).resolve_neg()
    return x2 if x2.dtype == torch.float16 else x2.half()


def _gradient(grad):
    """What autograd hands to a backward pass, as the kernels read it: float16 from a 16-byte boundary on.  (Of a part of a concatenation it is a view into the whole one's, at any place.)"""
    grad = grad.half().resolve_neg()
    return grad.clone() if grad.is_contiguous() and grad.data_ptr() % 16 else grad


class _InputGradient(torch.autograd.Function):
    """FPxLinear.forward, and the product with the weights the other way round.  What a backward pass needs is the weights alone."""

    @staticmethod
    def forward(ctx, x, layer):
        ctx.save_for_backward(layer.weight_native, layer.scales, layer.group_exps)
        ctx.format, ctx.in_features = (layer.exponent, layer.mantissa), layer.in_features
        return FPxLinear.forward(layer, x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, scales, exps = ctx.saved_tensors
        return ops.linear_input_grad_native(*ctx.format, _gradient(grad), weight, scales, ctx.in_features, group_exps=exps), None


class _GatedBlock(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block):
        preact = torch.empty(x.shape[0], 2 * block.out_features, dtype=torch.float32, device=x.device)
        y = block._values(x, preact)
        ctx.save_for_backward(preact, block.weight_native, block.scales, block.group_exps)
        ctx.format, ctx.in_features, ctx.activation = (block.exponent, block.mantissa), block.in_features, block.activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        preact, weight, scales, exps = ctx.saved_tensors
        return ops.gated_backward_native(*ctx.format, _gradient(grad), preact, weight, scales, ctx.in_features, ctx.activation, grad_preact=False, group_exps=exps)[0], None


_CROSSOVER, _CROSSOVER_LIBRARY = 32768, 3072   # FPxLinear.PREFILL_CROSSOVER as it is shipped, and the one without the wide tiles


class FPxLinear(torch.nn.Module):
    """y = x @ dequant(W)^T (+ bias) with W held in the native gfx950 layout.  Weights are buffers, not parameters:
    the layer is inference-only, like the kernels, but for input_gradient."""

    # True: an input that requires a gradient gets one, through the quantized weights (a frozen layer under trained adapters, prompts or layers below it).  Weights and bias have
    # none, and an input with a tangent (forward mode) is refused.  False, as it has always been: the kernels are no part of an autograd graph.
    input_gradient = False

    # Batch size from which dequantize + FP16 library GEMM is no slower than the mixed-input kernels, measured through this module at 4096^2, 8192^2, 28672x8192,
    # 8192x28672, 11008x4096, 1024x8192, 1024^2, 4608x4544 and 2560x18944, FP6 with row scales and FP5 with group exponents.  Kernel time / time of dequantization +
    # library GEMM: 0.33-0.99 at 3072 rows, 0.35-1.06 at 4096, 0.40-0.99 at 4100, 0.44-1.07 at 6144, 0.51-1.06 at 8192, 0.73-1.03 at 16384, 0.85-1.10 at 32768
    # (8192^2 at 4096 rows 369 us against 394, at 16384 1465 against 1464); with a bias, which the kernels add by themselves, 0.29-1.03 at 4096 and 0.58-0.96 at
    # 16384.  That is with the wide tiles, so on 256 CUs and with K up to 2^20; without them the two cross at 3072 rows.
    PREFILL_CROSSOVER = _CROSSOVER

    def __init__(self, in_features, out_features, exponent=3, mantissa=2, bias=None, split_k=None, dequant_above="auto", group_scales=False):
        """split_k: number of pieces of K, None for the heuristic's choice; under dequant_above="auto" it holds for less than 3072 rows.
        group_scales: the layer also holds one exponent byte per row and 128 columns (factor 1 until weights are loaded).
        dequant_above: batch size from which forward() dequantizes the weights to a temporary fp16 matrix on the GPU and calls
        the FP16 library GEMM instead (the temporary costs 2 bytes per weight for the duration of the call).  None never does; an
        integer sets the threshold; "auto" (default) is PREFILL_CROSSOVER rows, or 3072 where the wide tiles do not run.  Under "auto" an
        input of 3072 rows or more that the kernels cannot take as it is (_kernels_take: one that requires a gradient, say) also goes through
        the library.  A module that a version up to 138 pickled whole holds the number that "auto" was then, 3072."""
        super().__init__()
        self.dequant_above = dequant_above
        if out_features % 256 or in_features % 64:
            raise ValueError("FPxLinear needs out_features %% 256 == 0 and in_features %% 64 == 0")
        self.in_features, self.out_features = in_features, out_features
        self.exponent, self.mantissa = exponent, mantissa
        self.split_k = split_k
        self._split_cache = {}
        self.register_buffer("weight_native", torch.zeros(native_bytes(exponent, mantissa, out_features, in_features) // 4, dtype=torch.int32))
        self.register_buffer("scales", torch.ones(out_features, dtype=torch.float16))
        self.register_buffer("bias", bias)
        # per-group exponents (one byte per row and 128 columns, in the kernels' order), or None for row scales only
        self.register_buffer("group_exps", torch.full((group_exps_bytes(out_features, in_features),), 127, dtype=torch.uint8) if group_scales else None)

    @classmethod
    def from_raw(cls, raw_int32, scales, exponent=3, mantissa=2, bias=None, split_k=None):
        """raw_int32: the reference's raw weight tensor [OC, IC/32*x] (CPU); scales: float16 [OC]."""
        x = 1 + exponent + mantissa
        OC, IC = raw_int32.shape[0], raw_int32.shape[1] * 32 // x
        m = cls(IC, OC, exponent, mantissa, bias, split_k)
        m.weight_native.copy_(weight_prepacking_native_cpu(exponent, mantissa, raw_int32))
        m.scales.copy_(scales)
        return m

    @classmethod
    def from_prepacked(cls, packed_int32, scales, exponent=3, mantissa=2, bias=None, split_k=None):
        """packed_int32: output of weight_prepacking*_cpu (the reference layout), on CPU or GPU."""
        x = 1 + exponent + mantissa
        OC, IC = packed_int32.shape[0], packed_int32.shape[1] * 32 // x
        m = cls(IC, OC, exponent, mantissa, bias, split_k).to(packed_int32.device)
        m.weight_native.copy_(to_native(packed_int32, exponent, mantissa))
        m.scales.copy_(scales.to(packed_int32.device))
        return m

    @classmethod
    def from_float(cls, weight, exponent=3, mantissa=2, bias=None, split_k=None, group_scales=False):
        """Quantizes a float [OC, IC] weight row-wise (round to nearest even, absmax scales) and packs it; a weight that
        already lives on the GPU is quantized there (same bits as the host path).  group_scales=True adds a power-of-two
        factor per row and 128 columns (quant.quantize_groupwise), which the conversion instruction applies."""
        on_gpu = weight.device.type == "cuda" and weight.dtype in (torch.float16, torch.bfloat16, torch.float32)
        if group_scales and on_gpu:
            native, scales, gexp = weight_quantize_native_cuda(exponent, mantissa, weight.detach(), True)
            m = cls(weight.shape[1], weight.shape[0], exponent, mantissa, bias, split_k).to(weight.device)
            m.weight_native.copy_(native)
            m.scales.copy_(scales)
            m.group_exps = gexp
            return m
        if group_scales:
            codes, scales, exps = quant.quantize_groupwise(weight.detach().float().cpu().numpy(), exponent, mantissa)
            raw = torch.from_numpy(quant.pack_raw(codes, exponent, mantissa))
            m = cls.from_raw(raw, torch.from_numpy(scales), exponent, mantissa, bias, split_k)
            m.group_exps = pack_group_exps(torch.from_numpy(exps), weight.shape[0], weight.shape[1])
            return m.to(weight.device)
        if weight.device.type == "cuda" and weight.dtype in (torch.float16, torch.bfloat16, torch.float32):
            native, scales = weight_quantize_native_cuda(exponent, mantissa, weight.detach())
            m = cls(weight.shape[1], weight.shape[0], exponent, mantissa, bias, split_k).to(weight.device)
            m.weight_native.copy_(native)
            m.scales.copy_(scales)
            return m
        codes, scales = quant.quantize_rowwise(weight.detach().float().cpu().numpy(), exponent, mantissa)
        raw = torch.from_numpy(quant.pack_raw(codes, exponent, mantissa))
        return cls.from_raw(raw, torch.from_numpy(scales), exponent, mantissa, bias, split_k)

    @classmethod
    def fused(cls, layers, split_k=None):
        """One layer that computes several layers over the same input in a single launch (fused QKV, gate + up): its output
        is the concatenation of theirs along the feature axis.  Rows are independent in the native layout (16-row tiles
        are stored one after another), so fusing is a concatenation of the weight buffers, scales and biases."""
        layers = list(layers)
        first = layers[0]
        for l in layers:
            if (l.in_features, l.exponent, l.mantissa) != (first.in_features, first.exponent, first.mantissa):
                raise ValueError("fused layers must share in_features and the weight format")
            if (l.bias is None) != (first.bias is None):
                raise ValueError("fused layers must all have a bias or all have none")
            if l.weight_native.device != first.weight_native.device:
                raise ValueError("fused layers must live on one device")
            if (l.group_exps is None) != (first.group_exps is None):
                raise ValueError("fused layers must all have group exponents or all have none")
        bias = None if first.bias is None else torch.cat([l.bias for l in layers])
        m = cls(first.in_features, sum(l.out_features for l in layers), first.exponent, first.mantissa, bias, split_k)
        m = m.to(first.weight_native.device)
        m.weight_native.copy_(torch.cat([l.weight_native for l in layers]))
        m.scales.copy_(torch.cat([l.scales for l in layers]))
        if first.group_exps is not None:   # [row tile][K block][16][2] bytes: row tiles follow each other like the weights
            m.group_exps = torch.cat([l.group_exps for l in layers])
        return m

    def __getattr__(self, name):
        """nn.Module's, but that a buffer, of which a forward pass reads four, is looked for first (a call of a module with small kernels 7.9 -> 6.7 us)."""
        if name != "_buffers":   # (asked before nn.Module has made it, while a module is copied or unpickled)
            try:
                return self._buffers[name]
            except (KeyError, AttributeError):
                pass
        return super().__getattr__(name)

    def _wide_tiles(self, device):
        return self.in_features <= 1 << 20 and (device.type != "cuda" or torch.cuda.get_device_properties(device).multi_processor_count == MI355X_CUS)

    @property
    def dequant_above(self):
        """Rows from which forward() dequantizes an input that the kernels could take, on the weights' device; None: never."""
        if not self._auto:
            return self._rows
        return _AutoRows(self._rows if self._wide_tiles(self.weight_native.device) else _CROSSOVER_LIBRARY)

    @dequant_above.setter
    def dequant_above(self, rows):
        if isinstance(rows, str) and rows == "auto":   # (a subclass or a program with a PREFILL_CROSSOVER of its own means that number, whatever the device)
            rows = _AutoRows(_CROSSOVER) if self.PREFILL_CROSSOVER == _CROSSOVER else self.PREFILL_CROSSOVER
        self._auto = type(rows) is _AutoRows
        self._rows = _CROSSOVER if self._auto else rows

    def __setstate__(self, state):
        super().__setstate__(state)
        if "dequant_above" in self.__dict__:   # pickled whole when it was a plain attribute
            self.dequant_above = self.__dict__.pop("dequant_above")

    def _bias_in_kernel(self, x2):
        """Whether the kernels add the bias (to their float32 sums; otherwise a torch addition follows): a plain fp16 vector on the GPU that nothing
        differentiates or maps over."""
        b = self.bias
        return (b is not None and _values_only(b) and b.dtype == torch.float16 and b.shape == (self.out_features,) and b.is_contiguous() and b.device == x2.device)

    def _kernels_take(self, x2):
        """Whether a long prompt can leave torch.nn.functional.linear for the mixed-input kernels and nothing is lost: they are no part of an autograd graph, a
        trace or a transform, give fp16 whatever autocast would, and read contiguous rows at a 16-byte boundary; and only the wide tiles are faster."""
        kind = x2.device.type
        return (self._wide_tiles(x2.device) and _values_only(x2) and (not torch.is_autocast_enabled(kind) or torch.get_autocast_dtype(kind) == torch.float16)
                and (not x2.is_contiguous() or x2.data_ptr() % 16 == 0))

    def _with_adapters(self, x, adapters, index):
        if not isinstance(adapters, LowRankAdapters) or index is None:
            raise ValueError("adapters must be a LowRankAdapters, with an index for every row")
        if (adapters.in_features, adapters.out_features) != (self.in_features, self.out_features):
            raise ValueError("the adapters are for %d -> %d features, the layer has %d -> %d" % (adapters.in_features, adapters.out_features, self.in_features, self.out_features))
        bias, a, b, scaling = self.bias, _held(adapters, "lora_a"), _held(adapters, "lora_b"), _held(adapters, "scaling")
        if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad or scaling.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("a product with adapters has no gradient: call it under torch.no_grad()")
        x2 = _rows_of(x, self.in_features)
        if index.numel() != x2.shape[0] or (index.dim() != 1 and index.shape != x.shape[:-1]):
            raise ValueError("index must name an adapter for each of the %d rows, got %s" % (x2.shape[0], list(index.shape)))
        split = None if self._auto and x2.shape[0] >= _CROSSOVER_LIBRARY else self.split_k or None   # (as in forward: rows without an adapter have the layer's own bits)
        fused = bias if bias is not None and self._bias_in_kernel(x2) else None
        y = ops.adapter_forward_native(self.exponent, self.mantissa, x2, self.weight_native, self.scales, self.out_features, a, b, scaling,
                                       index.reshape(-1).contiguous(), split, group_exps=self.group_exps, bias=fused)
        if bias is not fused:
            y = y + bias
        return y.reshape(*x.shape[:-1], self.out_features)

    def forward(self, x, adapters=None, index=None):
        """adapters: a LowRankAdapters of this layer's shape, with index, int32, the slot of every row of x (-1: none).  With adapters the kernels take every batch, whatever
        dequant_above says."""
        if adapters is not None or index is not None:
            return self._with_adapters(x, adapters, index)
        # (two reshapes to the shapes at hand take 0.7 us each; a trace, whose sizes are no plain numbers, keeps them)
        shape = x.shape
        plain = type(x) is torch.Tensor and len(shape) == 2 and type(shape[1]) is int and shape[1] == self.in_features
        x2 = x if plain else x.reshape(-1, self.in_features)
        if x2.dtype != torch.float16:
            x2 = x2.half()
        if self.input_gradient and _differentiates(x):
            _refuse_unseen(x)
            if self.bias is not None and self.bias.requires_grad:
                raise ValueError("input_gradient is for a layer whose bias requires no gradient")
            y = _InputGradient.apply(x2, self)
            return y if plain else y.reshape(*shape[:-1], self.out_features)
        rows, n = self._rows, x2.shape[0]
        if rows is not None and (n >= rows or (self._auto and n >= _CROSSOVER_LIBRARY and not self._kernels_take(x2))):
            w16 = weight_dequant_native_cuda(self.exponent, self.mantissa, self.weight_native, self.scales, self.out_features, self.in_features,
                                             self.group_exps)
            y = torch.nn.functional.linear(x2, w16)
            del w16
            if self.bias is not None:
                y = y + self.bias
            return y if plain else y.reshape(*shape[:-1], self.out_features)
        if self.input_gradient:
            _refuse_unseen(x)
        sk = self.split_k
        if not sk or (self._auto and n >= _CROSSOVER_LIBRARY):   # the heuristic's answer per batch size is remembered: the layer is called once per token
            # (split_k is for the batches up to 3071 rows; the partial sums of a long prompt would take gigabytes)
            sk = self._split_cache.get(n)
            if sk is None:
                sk = self._split_cache[n] = heuristic_splitk_mi355x(self.out_features, n, self.in_features, MI355X_CUS, self.exponent, self.mantissa)
        bias = self.bias   # (a buffer, found by nn.Module.__getattr__ in half a microsecond: read once)
        OC, fused = self.out_features, bias if bias is not None and self._bias_in_kernel(x2) else None
        y = linear_forward_native(self.exponent, self.mantissa, x2, self.weight_native, self.scales, OC, sk, None, None, self.group_exps, fused)
        if bias is not fused:
            y = y + bias
        return y if plain else y.reshape(*shape[:-1], OC)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, format=e%dm%d" % (self.in_features, self.out_features, self.exponent, self.mantissa)


class FPxGatedLinear(torch.nn.Module):
    """y = act(x @ gate^T + bias_g) * (x @ up^T + bias_u): the first half of a gated feed-forward block in one launch, on native-layout weights that hold both matrices in pair order
    (ops.gate_up_pairs).  Differentiable in x; the weights are buffers and have no gradient."""

    def __init__(self, in_features, out_features, exponent=3, mantissa=2, activation="silu", bias=None, split_k=None, group_scales=False):
        """out_features: columns of y, the rows of gate and of up.  activation: "silu", "gelu" or "gelu_tanh".  bias: float16 [2 * out_features] in pair order.  split_k: number of
        pieces of K for less than 3072 rows, None for the heuristic's choice."""
        super().__init__()
        if out_features < 128 or out_features % 128 or in_features < 64 or in_features % 64:
            raise ValueError("FPxGatedLinear needs out_features %% 128 == 0 and in_features %% 64 == 0")
        ops._activation_code(activation)
        if bias is not None and (bias.dtype != torch.float16 or bias.shape != (2 * out_features,)):   # (inside the activation, so no addition can follow)
            raise ValueError("the bias of FPxGatedLinear must be float16 [%d], got %s %s" % (2 * out_features, str(bias.dtype).split(".")[-1], list(bias.shape)))
        self.in_features, self.out_features, self.exponent, self.mantissa = in_features, out_features, exponent, mantissa
        self.activation, self.split_k = activation, split_k
        self.register_buffer("weight_native", torch.zeros(native_bytes(exponent, mantissa, 2 * out_features, in_features) // 4, dtype=torch.int32))
        self.register_buffer("scales", torch.ones(2 * out_features, dtype=torch.float16))
        self.register_buffer("bias", bias)
        self.register_buffer("group_exps", torch.full((group_exps_bytes(2 * out_features, in_features),), 127, dtype=torch.uint8) if group_scales else None)

    @classmethod
    def from_layers(cls, gate, up, activation="silu", split_k=None):
        """From two FPxLinear of one shape and format: their bytes, in pair order."""
        for name in ("in_features", "out_features", "exponent", "mantissa"):
            if getattr(gate, name) != getattr(up, name):
                raise ValueError("gate and up must have the same %s" % name)
        for name in ("bias", "group_exps"):
            if (getattr(gate, name) is None) != (getattr(up, name) is None):
                raise ValueError("gate and up must both have %s or both have none" % name)
        F = gate.out_features
        m = cls(gate.in_features, F, gate.exponent, gate.mantissa, activation, None if gate.bias is None else ops.gate_up_pairs(gate.bias, up.bias), split_k)
        m = m.to(gate.weight_native.device)
        m.weight_native = ops.gate_up_pairs(gate.weight_native, up.weight_native, rows=F)
        m.scales = ops.gate_up_pairs(gate.scales, up.scales)
        if gate.group_exps is not None:
            m.group_exps = ops.gate_up_pairs(gate.group_exps, up.group_exps, rows=F)
        return m

    @classmethod
    def from_float(cls, gate, up, exponent=3, mantissa=2, activation="silu", bias=None, split_k=None, group_scales=False):
        """From two float [out_features, in_features] weights, quantized as FPxLinear.from_float does.  bias: (of gate, of up), float16."""
        both = FPxLinear.from_float(ops.gate_up_pairs(gate.detach(), up.detach()), exponent, mantissa, group_scales=group_scales)
        m = cls(gate.shape[1], gate.shape[0], exponent, mantissa, activation, None if bias is None else ops.gate_up_pairs(*bias), split_k).to(gate.device)
        m.weight_native, m.scales, m.group_exps = both.weight_native, both.scales, both.group_exps
        return m

    def _values(self, x2, preact=None):
        split = self.split_k or None if x2.shape[0] < _CROSSOVER_LIBRARY else None   # (as in FPxLinear: the partial sums of a long prompt would take gigabytes)
        return ops.gated_forward_native(self.exponent, self.mantissa, x2, _held(self, "weight_native"), _held(self, "scales"), 2 * self.out_features, self.activation, split, preact=preact,
                                        group_exps=_held(self, "group_exps"), bias=_held(self, "bias"))

    def forward(self, x):
        x2 = _rows_of(x, self.in_features)
        bias = _held(self, "bias")
        if bias is not None and bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("the bias of FPxGatedLinear has no gradient")
        y = _GatedBlock.apply(x2, self) if _differentiates(x) else self._values(x2)
        return y if x.dim() == 2 else y.reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, format=e%dm%d, activation=%s" % (self.in_features, self.out_features, self.exponent, self.mantissa, self.activation)


class LowRankAdapters(torch.nn.Module):
    """Slots for the low-rank adapters of many requests to one FPxLinear: layer(x, adapters, index) adds scaling * (x @ a^T) @ b^T to every row, with the a, b and scaling of the slot
    that the row's index names.  Buffers of fixed size, so a captured graph sees what set() and clear() write between its replays."""

    def __init__(self, in_features, out_features, slots, rank):
        """rank: the largest of any slot, up to 256; smaller ones are held with rows of zeros."""
        super().__init__()
        if out_features % 256 or in_features % 64:
            raise ValueError("LowRankAdapters needs out_features %% 256 == 0 and in_features %% 64 == 0")
        if slots < 1 or not 1 <= rank <= ops.MAX_RANK:
            raise ValueError("LowRankAdapters needs a slot at least, and a rank from 1 to %d" % ops.MAX_RANK)
        self.in_features, self.out_features, self.slots, self.rank = in_features, out_features, slots, (rank + 7) // 8 * 8
        self.register_buffer("lora_a", torch.zeros(slots, self.rank, in_features, dtype=torch.float16))
        self.register_buffer("lora_b", torch.zeros(slots, out_features, self.rank, dtype=torch.float16))
        self.register_buffer("scaling", torch.zeros(slots, dtype=torch.float32))

    def _apply(self, fn, *args, **kwargs):
        """nn.Module's, but that the buffers keep their types when a model around them is cast (the scalings are float32)."""
        before = dict(self._buffers)
        super()._apply(fn, *args, **kwargs)
        for name, t in before.items():
            if self._buffers[name].dtype != t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    @torch.no_grad()
    def set(self, slot, a, b, scaling=1.0):
        """a: [r, in_features], b: [out_features, r], r up to the rank.  For a fused layer lists of them, a pair for each part: their ranks add up, and a part's a reaches only its outputs."""
        if isinstance(a, (list, tuple)):
            if not a or len(a) != len(b) or any(p.dim() != 2 or q.dim() != 2 or p.shape[0] != q.shape[1] for p, q in zip(a, b)):
                raise ValueError("need an a [r, in_features] and a b [outputs, r] for each part")
            a, b = torch.cat(list(a)), torch.block_diag(*b)
        if not 0 <= slot < self.slots:
            raise ValueError("no slot %d among %d" % (slot, self.slots))
        r = a.shape[0]
        if a.shape != (r, self.in_features) or b.shape != (self.out_features, r) or r > self.rank:
            raise ValueError("need a [r, %d] and b [%d, r] with r up to %d, got %s and %s" % (self.in_features, self.out_features, self.rank, list(a.shape), list(b.shape)))
        self.clear(slot)
        self.lora_a[slot, :r].copy_(a)
        self.lora_b[slot, :, :r].copy_(b)
        self.scaling[slot] = scaling

    @torch.no_grad()
    def clear(self, slot):
        """Rows that name this slot are as without an adapter."""
        if not 0 <= slot < self.slots:
            raise ValueError("no slot %d among %d" % (slot, self.slots))
        self.lora_a[slot].zero_(), self.lora_b[slot].zero_(), self.scaling[slot].zero_()

    def extra_repr(self):
        return "in_features=%d, out_features=%d, slots=%d, rank=%d" % (self.in_features, self.out_features, self.slots, self.rank)


def save_native(path, native_int32, scales, exponent, mantissa, out_features, in_features, group_exps=None):
    """One weight matrix in the native layout: magic, little-endian uint32 header length, JSON header, native bytes, fp16 scales,
    then the packed group exponents if the weight has them."""
    nat = native_int32.detach().cpu().contiguous().numpy()
    sc = scales.detach().cpu().contiguous().numpy().astype(np.float16)
    if nat.nbytes != native_bytes(exponent, mantissa, out_features, in_features) or sc.shape != (out_features,):
        raise ValueError("buffers do not match the stated shape")
    ge = None
    if group_exps is not None:
        ge = group_exps.detach().cpu().contiguous().numpy()
        if ge.dtype != np.uint8 or ge.size != group_exps_bytes(out_features, in_features):
            raise ValueError("group_exps does not match the stated shape")
    header = json.dumps({"exponent": exponent, "mantissa": mantissa, "out_features": out_features, "in_features": in_features,
                         "layout": "native-v1", "native_bytes": int(nat.nbytes), "group_exps_bytes": 0 if ge is None else int(ge.size)}).encode()
    with open(path, "wb") as f:
        f.write(_MAGIC)
        f.write(struct.pack("<I", len(header)))
        f.write(header)
        f.write(nat.tobytes())
        f.write(sc.tobytes())
        if ge is not None:
            f.write(ge.tobytes())


def load_native(path):
    """Returns (native int32 tensor, float16 scales, header dict); the packed group exponents, if the file has them, are
    hdr["group_exps"] (uint8 tensor).  Plain binary parsing; nothing in the file is executed."""
    with open(path, "rb") as f:
        if f.read(len(_MAGIC)) != _MAGIC:
            raise ValueError("%s is not a native FPx weight file (or has another layout version)" % path)
        (hlen,) = struct.unpack("<I", f.read(4))
        if hlen > 1 << 16:
            raise ValueError("implausible header length")
        hdr = json.loads(f.read(hlen).decode())
        want = native_bytes(hdr["exponent"], hdr["mantissa"], hdr["out_features"], hdr["in_features"])
        if hdr.get("layout") != "native-v1" or hdr.get("native_bytes") != want:
            raise ValueError("header does not describe a native-v1 weight of that shape")
        nat = np.frombuffer(f.read(want), dtype=np.int32)
        sc = np.frombuffer(f.read(2 * hdr["out_features"]), dtype=np.float16)
        if nat.nbytes != want or sc.size != hdr["out_features"]:
            raise ValueError("file is truncated")
        gbytes = int(hdr.get("group_exps_bytes", 0))
        if gbytes:
            if gbytes != group_exps_bytes(hdr["out_features"], hdr["in_features"]):
                raise ValueError("header does not describe the group exponents of that shape")
            ge = np.frombuffer(f.read(gbytes), dtype=np.uint8)
            if ge.size != gbytes:
                raise ValueError("file is truncated")
            hdr["group_exps"] = torch.from_numpy(ge.copy())
    return torch.from_numpy(nat.copy()), torch.from_numpy(sc.copy()), hdr
