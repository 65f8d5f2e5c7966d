"""PyTorch glue over the C ABI: the custom operators ``kudnn_b200::linear``, ``::quantize`` and ``::grouped``, a drop-in module for
``nn.Linear`` and a feed-forward block of experts.

The reference reaches PyTorch through a patched build in which ``torch._C._set_kdnn_enabled(True)`` routes
``torch.nn.Linear`` to KuDNN (docs/zh/KuDNN_development_guide.md:1407-1486, 1748-1775).  Here the same dispatch point
is an ordinary ``torch.library`` operator: ``y = act(x . W^T + b) (+) residual`` on CUDA tensors, forward only (the
reference classes are FWD primitives too), with a fake (meta) implementation so that shape propagation, FakeTensor
tracing and ``torch.compile`` graph capture see the right output without touching the GPU.  All arithmetic happens in
libkudnn_b200.so; torch supplies the tensors, the current stream and the output allocation.
"""
import collections
import threading
from typing import Optional

import torch
from torch.multiprocessing.reductions import StorageWeakRef

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
ACTIVATIONS = {None: capi.ACT_NONE, "none": capi.ACT_NONE, "relu": capi.ACT_RELU, "silu": capi.ACT_SWISH,
               "swish": capi.ACT_SWISH, "gelu_tanh": capi.ACT_GELU_TANH, "gelu": capi.ACT_GELU_ERF,
               "gelu_erf": capi.ACT_GELU_ERF, "sigmoid": capi.ACT_SIGMOID, "tanh": capi.ACT_TANH}
RESIDUALS = {None: capi.RES_NONE, "none": capi.RES_NONE, "add": capi.RES_IDENTICAL, "ext": capi.RES_EXT,
             "mul": capi.RES_ELTWISE_MUL}

# Created primitives, keyed by everything the descriptor holds plus the weight's storage, address and version (a primitive
# pre-packs the weights it first sees and recognises them by pointer).  The weak reference kept beside a primitive holds
# the storage's identity, not its memory: as long as it exists no other storage has that identity, so weights that are
# allocated later where freed ones were never meet their packed copy.  Bounded: when full, the primitive used longest ago is
# dropped, and destroyed when no call of another thread uses it any more and after the lock is free again (that waits for the
# device); one whose launches a CUDA graph holds stays, however many they are.
_HANDLES = collections.OrderedDict()
_MAX_HANDLES = 128
_LOCK = threading.Lock()


def _handle(m, n, k, x, weight, bias, act, act_alpha, residual, res_op):
    code = _DTYPES[x.dtype]
    storage = weight.untyped_storage()
    key = (x.device.index, m, n, k, code, x.stride(-2) if x.dim() > 1 else k, storage._cdata, weight.data_ptr(), weight.stride(0),
           weight.stride(1), weight._version, None if bias is None else _DTYPES[bias.dtype], act, act_alpha, res_op)
    with _LOCK:
        entry = _HANDLES.get(key)
        if entry is not None:
            _HANDLES.move_to_end(key)
            return entry[0]
        desc = capi.make_desc(m, n, k, code, a_strides=(k, 1), b_strides=(weight.stride(1), weight.stride(0)),
                              has_bias=bias is not None, bias_dtype=None if bias is None else _DTYPES[bias.dtype], act=act,
                              act_alpha=act_alpha, res_op=res_op)
        lin = capi.Linear(desc)
        lin.prepack(weight, stream=torch.cuda.current_stream(x.device).cuda_stream)
        if len(_HANDLES) >= _MAX_HANDLES:
            oldest = next((old for old, (other, _) in _HANDLES.items() if other.graphs == 0), None)
            dropped = None if oldest is None else _HANDLES.pop(oldest)  # noqa: F841  (lives until this function has returned)
        _HANDLES[key] = (lin, StorageWeakRef(storage))
        return lin


def clear_cache():
    """Destroys every cached primitive (and the packed weight copies they own); graphs that hold calls of the operator
    must not be replayed afterwards."""
    with _LOCK:
        dropped = [entry[0] for cache in (_HANDLES, _GROUPED) for entry in cache.values()]
        _HANDLES.clear()
        _GROUPED.clear()
    for op in dropped:
        op.close()


def _run(x, x2, weight, bias, act, act_alpha, res2, res_op, gamma, m, n, k, out):
    lin = _handle(m, n, k, x2, weight, bias, act, act_alpha, res2, res_op)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    b = None if bias is None else bias.data_ptr()
    if res_op != capi.RES_NONE:
        lin.run(x2.data_ptr(), weight.data_ptr(), None, b, res2.data_ptr(), out.data_ptr(), gamma=gamma, stream=stream)
    else:
        lin.run(x2.data_ptr(), weight.data_ptr(), out.data_ptr(), b, stream=stream)


@torch.library.custom_op("kudnn_b200::linear", mutates_args=(), device_types="cuda")
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = 0,
           act_alpha: float = 1.0, residual: Optional[torch.Tensor] = None, res_op: int = 0,
           gamma: float = 1.0) -> torch.Tensor:
    """act(x . weight^T + bias), then (+) residual when res_op is given.  x [..., k], weight [n, k] as nn.Linear keeps
    it, bias [n], residual [..., n].  act / res_op are the KUDNN_B200_ACT_* / KUDNN_B200_RES_* codes."""
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise TypeError("kudnn_b200::linear takes float32 / float16 / bfloat16 tensors of one type")
    if weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError("kudnn_b200::linear: x [..., k] and weight [n, k] do not match")
    n, k = weight.shape
    x2 = x.reshape(-1, k)
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) != k):
        x2 = x2.contiguous()
    m = x2.shape[0]
    out = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    if m == 0:
        return out
    if bias is not None:
        bias = bias.contiguous()
    res2 = None
    if res_op != capi.RES_NONE:
        if residual is None or residual.shape != out.shape or residual.dtype != x.dtype:
            raise ValueError("kudnn_b200::linear: residual must have the output's shape and type")
        res2 = residual.contiguous()
    if x.device.index == torch.cuda.current_device():
        _run(x, x2, weight, bias, act, act_alpha, res2, res_op, gamma, m, n, k, out)
    else:
        with torch.cuda.device(x.device):
            _run(x, x2, weight, bias, act, act_alpha, res2, res_op, gamma, m, n, k, out)
    return out


@linear.register_fake
def _linear_fake(x, weight, bias=None, act=0, act_alpha=1.0, residual=None, res_op=0, gamma=1.0):
    return x.new_empty(x.shape[:-1] + (weight.shape[0],))


class Linear(torch.nn.Module):
    """``nn.Linear`` whose forward pass (inference) runs through ``kudnn_b200::linear``, optionally fused with an
    activation and a residual operand:  ``Linear.from_torch(layer, act="silu")(x)`` or ``(x, residual)``."""

    def __init__(self, in_features, out_features, bias=True, act=None, act_alpha=1.0, residual=None, gamma=1.0,
                 device=None, dtype=None):
        super().__init__()
        self.inner = torch.nn.Linear(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.act, self.act_alpha = ACTIVATIONS[act], float(act_alpha)
        self.res_op, self.gamma = RESIDUALS[residual], float(gamma)

    @classmethod
    def from_torch(cls, layer, act=None, act_alpha=1.0, residual=None, gamma=1.0):
        mod = cls.__new__(cls)
        torch.nn.Module.__init__(mod)
        mod.inner = layer
        mod.act, mod.act_alpha = ACTIVATIONS[act], float(act_alpha)
        mod.res_op, mod.gamma = RESIDUALS[residual], float(gamma)
        return mod

    def forward(self, x, residual=None):
        return torch.ops.kudnn_b200.linear(x, self.inner.weight, self.inner.bias, self.act, self.act_alpha, residual,
                                           self.res_op, self.gamma)


# ---- 8-bit floating point and experts

_OPERANDS = {torch.float16: capi.F16, torch.bfloat16: capi.BF16, torch.float8_e4m3fn: capi.E4M3}
_OFFSETS = {torch.int32: capi.S32, torch.int64: capi.S64}
# Created products by group: descriptors only, no weights and nothing of a call's tensors.  Bounded as _HANDLES; what was called while its
# stream was captured stays, since the graph must not outlive it, beyond the bound as well: a shape that graphs hold keeps its status word in
# device memory until clear_cache().
_GROUPED = collections.OrderedDict()
_MAX_GROUPED = 1024


def _pitch(k):
    return -(-k // 16) * 16


def _on(device):
    """The device of a call's tensors, current while it launches."""
    return torch.cuda.device(device)


def _quantized(x, rows, k, block_rows):
    """Uninitialised results of quantize beside x: q at a pitch of 16 bytes; the scales of one block of columns next to one another for
    activations, as the products read them, row-major for weights."""
    blocks_k, scale_rows = -(-k // capi.SCALE_BLOCK), -(-rows // block_rows)
    q = x.new_empty((rows, _pitch(k)), dtype=torch.float8_e4m3fn)[:, :k]
    if block_rows == 1:
        return q, x.new_empty((blocks_k, scale_rows), dtype=torch.float32).t()
    return q, x.new_empty((scale_rows, blocks_k), dtype=torch.float32)


@torch.library.custom_op("kudnn_b200::quantize", mutates_args=(), device_types="cuda")
def quantize(x: torch.Tensor, gate: bool = False, index: Optional[torch.Tensor] = None,
             block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows, k] -> (q, scale): e4m3 values and what to multiply them by.

    block_rows 1 (activations): a scale per row and 128 columns, scale [rows, ceil(k / 128)]; `gate`: of silu(x[:, :k]) * x[:, k:] for
    x [rows, 2 k]; `index` (int32): of the rows that it names, one outside of x gives zeros.  block_rows 128 (weights): a scale per
    128 x 128 block, scale [ceil(rows / 128), ceil(k / 128)].  Rows of q lie at a pitch of 16 bytes."""
    if x.dtype not in _DTYPES or x.dim() != 2:
        raise TypeError("kudnn_b200::quantize takes a float32 / float16 / bfloat16 matrix")
    if gate and x.shape[1] % 2 != 0:
        raise ValueError("kudnn_b200::quantize: a gate needs two halves of columns")
    if index is not None and (index.dtype != torch.int32 or index.dim() != 1 or index.device != x.device):
        raise ValueError("kudnn_b200::quantize: index is a vector of int32 on the device of x")
    if block_rows not in (1, capi.SCALE_BLOCK) or (block_rows != 1 and (gate or index is not None)):
        raise ValueError("kudnn_b200::quantize: blocks of 1 or 128 rows; a gate or an index goes with a scale per row")
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    rows, k = x.shape[0] if index is None else index.shape[0], x.shape[1] // 2 if gate else x.shape[1]
    q, scale = _quantized(x, rows, k, block_rows)
    if rows > 0:
        index = None if index is None else index.contiguous()
        desc = capi.make_quantize_desc(rows, k, _DTYPES[x.dtype], gate=gate, x_rows=x.shape[0], block_rows=block_rows,
                                       x_ld=x.stride(0) if x.shape[0] > 1 else x.shape[1], q_ld=_pitch(k), scale_strides=scale.stride())
        with _on(x.device):
            capi.quantize(desc, x, q, scale, index, stream=torch.cuda.current_stream(x.device).cuda_stream)
    return q, scale


@quantize.register_fake
def _quantize_fake(x, gate=False, index=None, block_rows=1):
    rows, k = x.shape[0] if index is None else index.shape[0], x.shape[1] // 2 if gate else x.shape[1]
    return _quantized(x, rows, k, block_rows)


def _grouped_handle(device, key, make):
    key = (device.index, key)
    with _LOCK:
        entry = _GROUPED.get(key)
        if entry is None:
            if len(_GROUPED) >= _MAX_GROUPED:
                oldest = next((old for old, (_, held) in _GROUPED.items() if not held), None)
                dropped = None if oldest is None else _GROUPED.pop(oldest)  # noqa: F841  (as in _handle)
            entry = _GROUPED[key] = [capi.Grouped(make()), False]
        else:
            _GROUPED.move_to_end(key)
        entry[1] = entry[1] or torch.cuda.is_current_stream_capturing()
        return entry[0]


@torch.library.custom_op("kudnn_b200::grouped", mutates_args=(), device_types="cuda")
def grouped(x: torch.Tensor, weight: torch.Tensor, offsets: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
            weight_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, act: int = 0, act_alpha: float = 1.0,
            out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[r] = act(x[r] . weight[g]^T + bias[g]) for offsets[g] <= r < offsets[g + 1]; rows that no group holds are zeros.

    x [rows, k], weight [groups, n, k] (or [n, k] without offsets), both float16, both bfloat16 or both float8_e4m3fn with x_scale
    [rows, ceil(k / 128)] and weight_scale [groups, ceil(n / 128), ceil(k / 128)]; offsets [groups + 1] int32 or int64 on the device;
    bias [groups, n].  The result is of out_dtype, by default bfloat16 for e4m3 operands and the operands' type otherwise."""
    if x.dtype not in _OPERANDS or weight.dtype != x.dtype:
        raise TypeError("kudnn_b200::grouped takes float16, bfloat16 or float8_e4m3fn tensors of one type")
    if weight.dim() == 2 and offsets is None:
        weight = weight.unsqueeze(0)
        weight_scale = None if weight_scale is None or weight_scale.dim() == 3 else weight_scale.unsqueeze(0)
        bias = None if bias is None or bias.dim() == 2 else bias.unsqueeze(0)
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2]:
        raise ValueError("kudnn_b200::grouped: x [rows, k] and weight [groups, n, k] do not match")
    (rows, k), (groups, n, _) = x.shape, weight.shape
    blocks = (-(-n // capi.SCALE_BLOCK), -(-k // capi.SCALE_BLOCK))
    if offsets is None:
        if groups != 1:
            raise ValueError("kudnn_b200::grouped: several groups need offsets")
    elif offsets.dtype not in _OFFSETS or offsets.shape != (groups + 1,) or offsets.device != x.device:
        raise ValueError("kudnn_b200::grouped: offsets are groups + 1 int32 or int64 values on the device of x")
    if x.dtype == torch.float8_e4m3fn:
        if x_scale is None or weight_scale is None or x_scale.shape != (rows, blocks[1]) or weight_scale.shape != (groups,) + blocks or \
                x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
            raise ValueError("kudnn_b200::grouped: e4m3 operands need float32 scales, one per row and 128 columns and one per 128 x 128 block")
    elif x_scale is not None or weight_scale is not None:
        raise ValueError("kudnn_b200::grouped: only e4m3 operands have scales")
    if bias is not None and (bias.dtype not in _DTYPES or bias.shape != (groups, n)):
        raise ValueError("kudnn_b200::grouped: bias is [groups, n]")
    out_dtype = out_dtype or (torch.bfloat16 if x.dtype == torch.float8_e4m3fn else x.dtype)
    if out_dtype not in _DTYPES:
        raise TypeError("kudnn_b200::grouped: results are float32, float16 or bfloat16")
    for other in (weight, x_scale, weight_scale, bias):
        if other is not None and other.device != x.device:
            raise ValueError("kudnn_b200::grouped: all tensors lie on one device")
    out = torch.empty((rows, n), dtype=out_dtype, device=x.device)
    if rows == 0:
        return out
    offsets = None if offsets is None else offsets.contiguous()
    key = (rows, n, k, groups, x.dtype, out_dtype, None if offsets is None else offsets.dtype, x.stride(), weight.stride(),
           None if x_scale is None else x_scale.stride(), None if weight_scale is None else weight_scale.stride(),
           None if bias is None else (bias.dtype, bias.stride()), act, act_alpha)

    def make():
        return capi.make_grouped_desc(
            rows, n, k, _OPERANDS[x.dtype], groups=groups, c_dtype=_DTYPES[out_dtype], offsets_dtype=0 if offsets is None else _OFFSETS[offsets.dtype],
            a_strides=x.stride(), b_strides=weight.stride(), a_scale_strides=None if x_scale is None else x_scale.stride(),
            b_scale_strides=None if weight_scale is None else weight_scale.stride(), has_bias=bias is not None,
            bias_dtype=None if bias is None else _DTYPES[bias.dtype], bias_strides=None if bias is None else bias.stride(), act=act,
            act_alpha=act_alpha)

    with _on(x.device):
        _grouped_handle(x.device, key, make).run(x, weight, out, offsets=offsets, a_scale=x_scale, b_scale=weight_scale, bias=bias,
                                                 stream=torch.cuda.current_stream(x.device).cuda_stream)
    return out


@grouped.register_fake
def _grouped_fake(x, weight, offsets=None, x_scale=None, weight_scale=None, bias=None, act=0, act_alpha=1.0, out_dtype=None):
    out_dtype = out_dtype or (torch.bfloat16 if x.dtype == torch.float8_e4m3fn else x.dtype)
    return x.new_empty((x.shape[0], weight.shape[-2]), dtype=out_dtype)


class Experts(torch.nn.Module):
    """Feed-forward block of experts (inference): every token goes to `top` experts, and what they answer is added up by weight.

        y[t] = sum over the token's experts e of p[t, e] * down[e](silu(gate[e](x[t])) * up[e](x[t]))

    p: softmax of the router's logits, the `top` largest made to sum to one.  gate_up [experts, 2 * ffn, hidden] holds gate's rows, then
    up's; down [experts, hidden, ffn].  With eight_bit the weights are kept as e4m3 with a scale per 128 x 128 block, the tokens are
    quantised on their way to the experts and the gated values between the two products.  Nothing is read back to the host."""

    def __init__(self, router, gate_up, down, top, eight_bit=False):
        super().__init__()
        if gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[1] != 2 * down.shape[2] or gate_up.shape[2] != down.shape[1] or \
                router.shape != (gate_up.shape[0], gate_up.shape[2]) or not 1 <= top <= gate_up.shape[0]:
            raise ValueError("Experts: router [experts, hidden], gate_up [experts, 2 * ffn, hidden] and down [experts, hidden, ffn] do not match")
        self.top, self.eight_bit = top, eight_bit
        self.register_buffer("router", router.float())
        for name, w in (("gate_up", gate_up), ("down", down)):
            if eight_bit:
                pairs = [torch.ops.kudnn_b200.quantize(w[e], block_rows=capi.SCALE_BLOCK) for e in range(w.shape[0])]
                packed = torch.empty(w.shape[:2] + (_pitch(w.shape[2]),), dtype=torch.float8_e4m3fn, device=w.device)
                for e, (q, _) in enumerate(pairs):
                    packed[e, :, :w.shape[2]].copy_(q)
                self.register_buffer(name, packed[:, :, :w.shape[2]])
                self.register_buffer(name + "_scale", torch.stack([s for _, s in pairs]))
            else:
                self.register_buffer(name, w)

    def _apply(self, fn, recurse=True):
        """Moves of the module (``to``, ``cuda``, ``half`` ...): the router, scales and e4m3 weights go along but keep their types, and the
        weights the pitch that the products read in place."""
        names = ("router", "gate_up", "gate_up_scale", "down", "down_scale") if self.eight_bit else ("router",)
        kept = {name: self._buffers[name] for name in names}
        self._buffers.update(dict.fromkeys(names))
        super()._apply(fn, recurse)
        for name, t in kept.items():
            e4m3 = t.dtype == torch.float8_e4m3fn
            if e4m3:  # with the bytes between the rows
                bits = torch.as_strided(t, t.shape[:2] + (t.stride(1),), t.stride(), t.storage_offset()).view(torch.uint8)
            else:
                bits = t.view(torch.int32)
            moved = fn(bits)
            if moved.dtype != bits.dtype:
                moved = bits.to(moved.device)
            self._buffers[name] = moved.view(t.dtype)[:, :, :t.shape[2]] if e4m3 else moved.view(t.dtype)
        return self

    @torch.no_grad()
    def forward(self, x):
        tokens = x.reshape(-1, x.shape[-1])
        count, experts = tokens.shape[0], self.router.shape[0]
        ops = torch.ops.kudnn_b200
        p, chosen = torch.topk(torch.softmax(ops.linear(tokens.float(), self.router), dim=1), self.top, dim=1)
        p = p / p.sum(dim=1, keepdim=True)
        # rows sorted by expert; a stable sort keeps the tokens of an expert in order
        owner, order = torch.sort(chosen.reshape(-1), stable=True)
        offsets = torch.searchsorted(owner, torch.arange(experts + 1, device=x.device, dtype=owner.dtype)).to(torch.int32)
        source = torch.div(order, self.top, rounding_mode="floor").to(torch.int32)
        if self.eight_bit:
            q, scale = ops.quantize(tokens, False, source)
            h = ops.grouped(q, self.gate_up, offsets, scale, self.gate_up_scale, out_dtype=x.dtype)
            q, scale = ops.quantize(h, True)
            y = ops.grouped(q, self.down, offsets, scale, self.down_scale, out_dtype=x.dtype)
        else:
            h = ops.grouped(tokens[source.long()], self.gate_up, offsets)
            gate, up = h.float().chunk(2, dim=1)
            y = ops.grouped((torch.nn.functional.silu(gate) * up).to(x.dtype), self.down, offsets)
        back = torch.empty_like(order)
        back[order] = torch.arange(order.shape[0], device=x.device)
        y = (y[back].view(count, self.top, tokens.shape[1]).float() * p[:, :, None]).sum(dim=1)
        return y.to(x.dtype).view(x.shape)
