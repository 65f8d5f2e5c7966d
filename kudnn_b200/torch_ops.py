"""PyTorch glue over the C ABI: the custom operators ``kudnn_b200::linear``, ``::quantize``, ``::grouped``, ``::layernorm``, ``::route`` and
``::experts``, drop-in modules for ``nn.Linear`` and ``nn.LayerNorm`` and a feed-forward block of experts.

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


# ---- a router and a block of experts for few tokens

SCORES = {"softmax": capi.SCORE_SOFTMAX, "sigmoid": capi.SCORE_SIGMOID}
MOST_FEW_TOKENS, MOST_FEW_TOP = 64, 16


@torch.library.custom_op("kudnn_b200::route", mutates_args=(), device_types="cuda")
def route(x: torch.Tensor, router: torch.Tensor, top: int, bias: Optional[torch.Tensor] = None, score: str = "softmax", normalise: bool = True,
          scale: float = 1.0, nan_first: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """x [tokens, hidden], router [experts, hidden] -> (weights [tokens, top] float32, ids [tokens, top] int32), the largest score first.

    Scores are a softmax or a sigmoid of x . router^T, computed in 64 bits.  bias [experts] float32 is added to them for the choice alone; minus
    infinity takes an expert out.  With `normalise` a token's weights are divided by their sum, then multiplied by `scale`.  Places that no
    expert is left for have the id -1 and the weight 0.  An expert whose score is NaN takes no part, or with `nan_first` comes before all others
    with a weight of NaN, as in torch.topk."""
    if x.dtype not in _DTYPES or router.dtype not in _DTYPES:
        raise TypeError("kudnn_b200::route takes float32 / float16 / bfloat16 tokens and routers")
    if x.dim() != 2 or router.dim() != 2 or x.shape[1] != router.shape[1] or router.device != x.device:
        raise ValueError("kudnn_b200::route: x [tokens, hidden] and router [experts, hidden] on one device do not match")
    if score not in SCORES:
        raise ValueError("kudnn_b200::route: scores are softmax or sigmoid")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != router.shape[:1] or bias.device != x.device):
        raise ValueError("kudnn_b200::route: bias is a float32 vector of the experts on the device of x")
    x, router = [t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous() for t in (x, router)]
    tokens = x.shape[0]
    weights = torch.empty((tokens, top), dtype=torch.float32, device=x.device)
    ids = torch.empty((tokens, top), dtype=torch.int32, device=x.device)
    desc = capi.make_route_desc(tokens, router.shape[0], x.shape[1], top, _DTYPES[x.dtype], router_dtype=_DTYPES[router.dtype], score=SCORES[score],
                                normalise=normalise, scale=scale, x_ld=x.stride(0), w_ld=router.stride(0), nan_first=nan_first)
    with _on(x.device):
        capi.route(desc, x, router, weights, ids, None if bias is None else bias.contiguous(), stream=torch.cuda.current_stream(x.device).cuda_stream)
    return weights, ids


@route.register_fake
def _route_fake(x, router, top, bias=None, score="softmax", normalise=True, scale=1.0, nan_first=False):
    return x.new_empty((x.shape[0], top), dtype=torch.float32), x.new_empty((x.shape[0], top), dtype=torch.int32)


@torch.library.custom_op("kudnn_b200::experts", mutates_args=(), device_types="cuda")
def experts(x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, gate_up: torch.Tensor, down: torch.Tensor,
            gate_up_scale: Optional[torch.Tensor] = None, down_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum over j of weights[t, j] * down[e](silu(gate[e](x[t])) * up[e](x[t])), e = ids[t, j], for at most 64 tokens.

    x [tokens, hidden] float16 or bfloat16; weights float32 and ids int32 [tokens, top] as route gives them; gate_up [experts, 2 ffn, hidden] and
    down [experts, hidden, ffn] of x's type, or float8_e4m3fn with float32 scales per 128 x 128."""
    if x.dtype not in (torch.float16, torch.bfloat16) or gate_up.dtype not in (x.dtype, torch.float8_e4m3fn) or down.dtype != gate_up.dtype:
        raise TypeError("kudnn_b200::experts takes float16 or bfloat16 tokens and weights of that type or of float8_e4m3fn")
    if x.dim() != 2 or gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[1] % 2 != 0 or \
            down.shape != (gate_up.shape[0], gate_up.shape[2], gate_up.shape[1] // 2) or x.shape[1] != gate_up.shape[2]:
        raise ValueError("kudnn_b200::experts: x [tokens, hidden], gate_up [experts, 2 * ffn, hidden] and down [experts, hidden, ffn] do not match")
    (tokens, hidden), (count, ffn) = x.shape, (gate_up.shape[0], down.shape[2])
    if weights.dtype != torch.float32 or ids.dtype != torch.int32 or weights.dim() != 2 or weights.shape != ids.shape or ids.shape[0] != tokens:
        raise ValueError("kudnn_b200::experts: weights float32 and ids int32 are [tokens, top]")
    inner, outer = -(-ffn // capi.SCALE_BLOCK), -(-hidden // capi.SCALE_BLOCK)
    shapes = ((count, -(-2 * ffn // capi.SCALE_BLOCK), outer), (count, outer, inner))
    for scale, shape in zip((gate_up_scale, down_scale), shapes):
        if (scale is not None) != (gate_up.dtype == torch.float8_e4m3fn) or (scale is not None and (scale.dtype != torch.float32 or scale.shape != shape)):
            raise ValueError("kudnn_b200::experts: e4m3 weights need float32 scales per 128 x 128, others take none")
    for other in (weights, ids, gate_up, down, gate_up_scale, down_scale):
        if other is not None and other.device != x.device:
            raise ValueError("kudnn_b200::experts: all tensors lie on one device")
    if x.stride(1) != 1 and hidden > 1:
        x = x.contiguous()
    y = torch.empty((tokens, hidden), dtype=x.dtype, device=x.device)
    desc = capi.make_experts_desc(tokens, hidden, ffn, count, ids.shape[1], _DTYPES[x.dtype], weight_dtype=_OPERANDS[gate_up.dtype],
                                  x_ld=x.stride(0) if tokens > 1 else hidden, gate_up_strides=gate_up.stride(), down_strides=down.stride(),
                                  gate_up_scale_strides=None if gate_up_scale is None else gate_up_scale.stride(),
                                  down_scale_strides=None if down_scale is None else down_scale.stride())
    size = capi.experts_workspace(desc)
    # scratch of this call alone: calls on other streams and in graphs have theirs
    space = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
    with _on(x.device):
        capi.experts(desc, x, weights.contiguous(), ids.contiguous(), gate_up, down, y, space, size, gate_up_scale, down_scale,
                     stream=torch.cuda.current_stream(x.device).cuda_stream)
    return y


@experts.register_fake
def _experts_fake(x, weights, ids, gate_up, down, gate_up_scale=None, down_scale=None):
    return x.new_empty(x.shape)


class Experts(torch.nn.Module):
    """Feed-forward block of experts (inference): every token goes to `top` experts, and what they answer is added up by weight.

        y[t] = sum over the token's experts e of p[t, e] * down[e](silu(gate[e](x[t])) * up[e](x[t]))

    p: softmax of the router's logits, the `top` largest made to sum to one.  gate_up [experts, 2 * ffn, hidden] holds gate's rows, then
    up's; down [experts, hidden, ffn].  With eight_bit the weights are kept as e4m3 with a scale per 128 x 128 block, the tokens are
    quantised on their way to the experts and the gated values between the two products.  Nothing is read back to the host.

    few: calls of 16-bit tokens, at most so many (64, and a top of 16, at most), go through ``route`` and ``experts`` instead, three launches in
    all, which read each chosen expert's weights once and quantise nothing but the weights.  8 suits large experts (4096 x 2048), up to 64 small ones
    (1024 x 704).  Whether a wait in those kernels gave up, ``kudnn_b200.experts_check`` tells; the module does not ask."""

    def __init__(self, router, gate_up, down, top, eight_bit=False, few=0):
        super().__init__()
        if gate_up.dim() != 3 or down.dim() != 3 or gate_up.shape[1] != 2 * down.shape[2] or gate_up.shape[2] != down.shape[1] or \
                router.shape != (gate_up.shape[0], gate_up.shape[2]) or not 1 <= top <= gate_up.shape[0]:
            raise ValueError("Experts: router [experts, hidden], gate_up [experts, 2 * ffn, hidden] and down [experts, hidden, ffn] do not match")
        if not 0 <= few <= MOST_FEW_TOKENS or (few > 0 and top > MOST_FEW_TOP):
            raise ValueError("Experts: few is at most 64, and with it top at most 16")
        self.top, self.eight_bit, self.few = top, eight_bit, few
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
        if 0 < self.few and count <= self.few and x.dtype in (torch.float16, torch.bfloat16) and (self.eight_bit or self.gate_up.dtype == x.dtype):
            p, chosen = ops.route(tokens, self.router, self.top, nan_first=True)  # a token without a softmax stays visible, as below
            scales = (self.gate_up_scale, self.down_scale) if self.eight_bit else (None, None)
            return ops.experts(tokens, p, chosen, self.gate_up, self.down, *scales).view(x.shape)
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


# ---- layer normalisation


def _rows(t):
    """[..., axis] as rows with contiguous elements."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _layernorm_desc(x, param, has_scale, has_shift, eps, dy=None):
    rows, axis = x.shape

    def pitch(t):
        return t.stride(0) if rows > 1 else axis

    return capi.make_layernorm_desc(rows, axis, _DTYPES[x.dtype], param_dtype=_DTYPES[x.dtype if param is None else param.dtype],
                                    has_scale=has_scale, has_shift=has_shift, eps=eps, x_ld=pitch(x), dy_ld=None if dy is None else pitch(dy))


def _check_layernorm(x, scale, shift):
    if x.dtype not in _DTYPES or x.dim() < 1 or x.shape[-1] == 0:
        raise TypeError("kudnn_b200::layernorm takes float32 / float16 / bfloat16 rows")
    for t in (scale, shift):
        if t is not None and (t.shape != x.shape[-1:] or t.dtype not in (x.dtype, torch.float32) or t.device != x.device):
            raise ValueError("kudnn_b200::layernorm: scale and shift are vectors of the last axis, float32 or of x's type, on its device")
    if scale is not None and shift is not None and scale.dtype != shift.dtype:
        raise ValueError("kudnn_b200::layernorm: scale and shift are of one type")


@torch.library.custom_op("kudnn_b200::layernorm", mutates_args=(), device_types="cuda")
def layernorm(x: torch.Tensor, scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
              eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(x - mean) / sqrt(variance + eps) * scale + shift over the last axis, with the mean and the variance of every row (float32).

    scale, shift: float32 or of x's type.  Differentiable with respect to x, scale and shift (the first result's gradient only)."""
    _check_layernorm(x, scale, shift)
    rows = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, variance = [torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) for _ in range(2)]
    desc = _layernorm_desc(rows, scale if scale is not None else shift, scale is not None, shift is not None, eps)
    with _on(x.device):
        capi.layernorm(desc, rows, y, None if scale is None else scale.contiguous(), None if shift is None else shift.contiguous(), mean, variance,
                       stream=torch.cuda.current_stream(x.device).cuda_stream)
    return y, mean, variance


@layernorm.register_fake
def _layernorm_fake(x, scale=None, shift=None, eps=1e-5):
    return x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("kudnn_b200::layernorm_backward", mutates_args=(), device_types="cuda")
def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, scale: Optional[torch.Tensor], mean: torch.Tensor, variance: torch.Tensor,
                       eps: float, param_dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of layernorm's x, scale and shift, the latter two of param_dtype."""
    _check_layernorm(x, scale, None)
    if dy.shape != x.shape or dy.dtype != x.dtype or mean.shape != x.shape[:-1] or variance.shape != mean.shape or \
            mean.dtype != torch.float32 or variance.dtype != torch.float32 or any(t.device != x.device for t in (dy, mean, variance)):
        raise ValueError("kudnn_b200::layernorm_backward: dy, mean and variance do not match x or lie on another device")
    if param_dtype not in (x.dtype, torch.float32) or (scale is not None and scale.dtype != param_dtype):
        raise ValueError("kudnn_b200::layernorm_backward: scale and the gradients are of one type, float32 or that of x")
    rows, dy_rows = _rows(x), _rows(dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dscale, dshift = [torch.empty(x.shape[-1:], dtype=param_dtype, device=x.device) for _ in range(2)]
    desc = _layernorm_desc(rows, dscale, scale is not None, False, eps, dy=dy_rows)
    size = capi.layernorm_backward_workspace(desc)
    space = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
    with _on(x.device):
        capi.layernorm_backward(desc, rows, dy_rows, None if scale is None else scale.contiguous(), mean.contiguous(), variance.contiguous(), dx, dscale,
                                dshift, space, size, stream=torch.cuda.current_stream(x.device).cuda_stream)
    return dx, dscale, dshift


@layernorm_backward.register_fake
def _layernorm_backward_fake(dy, x, scale, mean, variance, eps, param_dtype):
    return x.new_empty(x.shape), x.new_empty(x.shape[-1:], dtype=param_dtype), x.new_empty(x.shape[-1:], dtype=param_dtype)


def _layernorm_context(ctx, inputs, output):
    x, scale, shift, eps = inputs
    _, mean, variance = output
    ctx.mark_non_differentiable(mean, variance)
    ctx.save_for_backward(x, scale, mean, variance)
    ctx.eps, ctx.param_dtype, ctx.with_scale, ctx.with_shift = eps, (scale if scale is not None else shift if shift is not None else x).dtype, \
        scale is not None, shift is not None


def _layernorm_gradient(ctx, dy, _mean, _variance):
    x, scale, mean, variance = ctx.saved_tensors
    dx, dscale, dshift = torch.ops.kudnn_b200.layernorm_backward(dy, x, scale, mean, variance, ctx.eps, ctx.param_dtype)
    return dx, dscale if ctx.with_scale else None, dshift if ctx.with_shift else None, None


layernorm.register_autograd(_layernorm_gradient, setup_context=_layernorm_context)


class LayerNorm(torch.nn.Module):
    """``nn.LayerNorm`` over the last axis through ``kudnn_b200::layernorm``, forward and backward:  ``LayerNorm.from_torch(layer)(x)``.

    As with every autograd function of torch: while a backward pass is captured into a CUDA graph, no eager graph of the same parameters may be
    alive (delete its results first), or torch's own accumulation of gradients waits for a stream that is not captured."""

    def __init__(self, axis, eps=1e-5, bias=True, device=None, dtype=None):
        super().__init__()
        self.inner = torch.nn.LayerNorm(axis, eps=eps, bias=bias, device=device, dtype=dtype)

    @classmethod
    def from_torch(cls, layer):
        if len(layer.normalized_shape) != 1:
            raise ValueError("LayerNorm: one axis, the last")
        mod = cls.__new__(cls)
        torch.nn.Module.__init__(mod)
        mod.inner = layer
        return mod

    def forward(self, x):
        return torch.ops.kudnn_b200.layernorm(x, self.inner.weight, self.inner.bias, self.inner.eps)[0]
