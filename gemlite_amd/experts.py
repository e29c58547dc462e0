"""Mixture of experts on quantised weights: routing, and products grouped by expert.

No counterpart in the reference, which has one layer object per matrix: a mixture-of-experts block would be one launch per
expert and a host synchronisation for the row counts.  Here the rows of all experts go through one launch per matrix,
and the row counts stay on the GPU.

    plan = route_experts(logits, top_k)              # who goes where
    h = gate_up.forward_gated(x, plan)                # silu(x W_gate) * (x W_up), rows sorted by expert
    y = down.forward_combined(h, plan)                # weighted sum of every token's experts

``GemLiteExperts`` stacks packed ``GemLiteLinear`` layers of one kind; ``GemLiteMoE`` is the three lines above as a module.
As everywhere in this package the products have no backward pass: outputs carry no gradient.
"""
import logging
import threading
from typing import List, NamedTuple, Optional

import torch
from torch import Tensor

from . import _ext
from .core import GemLiteLinear
from .dtypes import DType, DTYPE_TO_TORCH, TORCH_TO_DTYPE

logger = logging.getLogger(__name__)

SCORINGS = {"softmax": 0, "sigmoid": 1}
_ROWS, _GATED, _COMBINED = 0, 1, 2


class ExpertPlan(NamedTuple):
    """Which experts every token goes to, and the (token, slot) pairs sorted by expert.

    ``weights`` [T, k] fp32 and ``expert_ids`` [T, k] int32 (-1 or another id outside ``0 .. E - 1``: no expert); ``offsets`` [E + 1] int32: rows
    ``offsets[e] .. offsets[e + 1] - 1`` of the sorted rows are expert ``e``'s, rows from ``offsets[E]`` on have none;
    ``order`` [T k] int32: flat index ``token * k + slot`` of every sorted row; ``places`` [T, k] int32: sorted row of
    every pair.
    """

    weights: Tensor
    expert_ids: Tensor
    offsets: Tensor
    order: Tensor
    places: Tensor


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------
def _empty_plan(like, T, k, E, apart=False):
    """(ids, offsets, order, places): views of one allocation (the kernels address them element by element), or ``apart``."""
    _ext._route_need(T, E, k)  # (refuses sizes that no plan can have)
    n = T * k
    if apart:
        return tuple(like.new_empty(shape, dtype=torch.int32) for shape in ((T, k), (E + 1,), (n,), (T, k)))
    ints = like.new_empty(3 * n + E + 1, dtype=torch.int32)
    return (ints.as_strided((T, k), (k, 1), 0), ints.as_strided((E + 1,), (1,), 3 * n), ints.as_strided((n,), (1,), n),
            ints.as_strided((T, k), (k, 1), 2 * n))


def route_experts(logits: Tensor, top_k: int, scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0) -> ExpertPlan:
    """The ``top_k`` largest of every row of ``logits`` [T, E] (fp32, fp16 or bf16) and the plan of these choices.

    Largest first, ties to the lower expert; NaN and -inf are never chosen: where a row has fewer than ``top_k`` others
    the remaining slots get id -1 and weight 0.  Weights are ``scoring`` ("softmax" or "sigmoid") of the logits in fp32,
    with ``renormalize`` divided by their sum over the chosen ones, times ``scale``.
    """
    if route_experts_op is not None and torch.compiler.is_compiling():
        return ExpertPlan(*route_experts_op(logits, top_k, scoring, renormalize, scale))
    return _route_experts(logits, top_k, scoring, renormalize, scale)


def _route_experts(logits, top_k, scoring, renormalize, scale, apart=False):
    if logits.dim() != 2:
        raise ValueError(f"logits: expected [tokens, experts], got shape {tuple(logits.shape)}")
    if scoring not in SCORINGS:
        raise ValueError(f"scoring: expected one of {sorted(SCORINGS)}, got {scoring!r}")
    _ext._require_cuda(logits)
    T, E = logits.shape
    if not 1 <= top_k <= min(E, 64):
        raise ValueError(f"top_k: expected 1 .. {min(E, 64)}, got {top_k}")
    if logits.stride(1) != 1 or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    weights = logits.new_empty((T, top_k), dtype=torch.float32)
    ids, offsets, order, places = _empty_plan(logits, T, top_k, E, apart)
    _ext.route_experts(logits, top_k, SCORINGS[scoring], renormalize, scale, weights, ids, offsets, order, places)
    return ExpertPlan(weights, ids, offsets, order, places)


def plan_experts(expert_ids: Tensor, weights: Tensor, num_experts: int) -> ExpertPlan:
    """The plan of choices made elsewhere: ``expert_ids`` [T, k] (ids outside ``0 .. num_experts - 1``, as those of another
    rank's experts, mean no expert) and ``weights`` [T, k]."""
    if expert_ids.dim() != 2 or expert_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_ids: expected [tokens, slots] int32 or int64, got {tuple(expert_ids.shape)} {expert_ids.dtype}")
    if weights.shape != expert_ids.shape or weights.device != expert_ids.device:
        raise ValueError(f"weights: expected shape {tuple(expert_ids.shape)} on {expert_ids.device}, got {tuple(weights.shape)} on {weights.device}")
    _ext._require_cuda(expert_ids)
    if expert_ids.dtype == torch.int64:
        # (ids that 32 bits cannot hold are no expert either)
        expert_ids = expert_ids.clamp(-1, 2 ** 31 - 1)
    ids = expert_ids.to(torch.int32).contiguous()
    T, k = ids.shape
    _, offsets, order, places = _empty_plan(ids, T, k, int(num_experts))
    _ext.plan_experts(ids, num_experts, offsets, order, places)
    return ExpertPlan(weights.to(torch.float32).contiguous(), ids, offsets, order, places)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _plan_tensor(name, t, shape, dtype, device):
    if tuple(t.shape) != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous {dtype} {shape} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _weights_of(tensor_args, meta_args):
    """Shapes of stacked experts: (E, N, K), with the layout of every expert checked."""
    W_q, scales, zeros = tensor_args[0], tensor_args[1], tensor_args[2]
    nbits, group, e = int(meta_args[1]), int(meta_args[2]), int(meta_args[4])
    if W_q.dim() != 3:
        raise ValueError(f"W_q: expected [experts, K / {e}, N], got shape {tuple(W_q.shape)}")
    E, rows, N = W_q.shape
    K = rows * e
    inner = (N, 1) if nbits < 8 else (1, K)
    want = {4: (torch.int32,), 8: (torch.float8_e4m3fn,), 16: (torch.float16, torch.bfloat16)}.get(nbits, ())
    if W_q.dtype not in want:
        raise NotImplementedError(f"experts of {nbits}-bit weights stored as {W_q.dtype} are not built "
                                  "(4-bit codes in int32 words, float8_e4m3fn, 16-bit floats)")
    if W_q.stride()[1:] != inner or (E > 1 and W_q.stride(0) < rows * N):
        raise ValueError(f"W_q: strides {W_q.stride()} of {tuple(W_q.shape)}; every expert has to be laid out with strides {inner}")
    if nbits == 4:
        if group <= 0 or K % group:
            raise ValueError(f"group_size {group} does not divide K={K}")
        for name, t in (("scales", scales), ("zeros", zeros)):
            if name == "zeros" and int(meta_args[10]) == 2:
                continue
            if tuple(t.shape) != (E, K // group, N) or not t.is_contiguous() or t.dtype != scales.dtype:
                raise ValueError(f"{name}: expected contiguous {scales.dtype} {(E, K // group, N)}, got {t.dtype} {tuple(t.shape)}")
    elif nbits == 8:
        want_s = (E, K // 128, (N + 127) // 128)
        if tuple(scales.shape) != want_s or not scales.is_contiguous() or scales.dtype != torch.float32:
            raise ValueError(f"scales: expected contiguous float32 {want_s}, got {scales.dtype} {tuple(scales.shape)}")
    return E, N, K


# Filling and checking a gla_experts_args takes longer than a decode-sized launch, so a filled struct is kept per kind of
# call (shapes, strides, types, devices, modes: never addresses or objects) and later calls of the kind only set the
# addresses.  Entries are per thread: the struct is rewritten in place on every call.
_PREPARED = {}
_PREPARED_LIMIT = 4096
_thread_id = threading.get_ident


def _prepare(mode, x, fits, bias, tensor_args, meta_args, offsets, plan, tile_config):
    """Checks a call and returns (struct, workspace bytes, shape of the output, its type)."""
    W_q, scales, zeros = tensor_args[0], tensor_args[1], tensor_args[2]
    meta = [int(v) for v in meta_args]
    (scaled, nbits, group, _, e, _, out_code, _, _, csm, wgm, _) = meta
    if x.dim() != 2:
        raise ValueError(f"x: expected [rows, K], got shape {tuple(x.shape)}")
    _ext._require_cuda(x, W_q, bias, offsets)
    E, N, K = _weights_of(tensor_args, meta)
    if x.shape[1] != K:
        raise ValueError(f"x: rows of {x.shape[1]} values for experts with K={K}")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"experts take fp16 or bf16 activations, got {x.dtype}")
    if nbits == 16 and W_q.dtype != x.dtype:
        raise NotImplementedError(f"16-bit experts of {W_q.dtype} take activations of that type, got {x.dtype}")
    for name, t in (("W_q", W_q), ("scales", scales), ("zeros", zeros), ("bias", bias)):
        if t is not None and t.numel() > 0 and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    device = x.device

    sizes = (E, N, K, x.shape[0]) if plan is None else (E, N, K, x.shape[0], plan.places.numel(), *plan.places.shape)
    if max(sizes) >= 2 ** 31:
        raise ValueError(f"sizes {sizes}: the library takes 32-bit integers")
    a = _ext.ExpertsArgs()
    a.mode = mode
    a.E, a.N, a.K = E, N, K
    a.W_nbits, a.group_size, a.elements_per_sample = nbits, group, e
    a.channel_scale_mode, a.W_group_mode, a.output_dtype = csm, wgm, out_code
    a.tile_config = tile_config
    a.offsets = _plan_tensor("offsets", offsets, (E + 1,), torch.int32, device)
    rows = x.shape[0]
    out_rows, out_cols = rows, N
    if plan is not None:
        T, k = plan.places.shape
        out_rows = T if mode == _COMBINED else T * k
        if rows != (T if mode == _GATED else T * k):
            raise ValueError(f"x: {rows} rows for a plan of {T} tokens with {k} experts each")
        a.T, a.top_k, a.R = T, k, T * k
        if mode == _GATED:
            a.order = _plan_tensor("plan.order", plan.order, (T * k,), torch.int32, device)
            out_cols = N // 2
        else:
            a.places = _plan_tensor("plan.places", plan.places, (T, k), torch.int32, device)
            a.weights = _plan_tensor("plan.weights", plan.weights, (T, k), torch.float32, device)
    else:
        a.R = rows
    if bias is not None:
        a.bias = _plan_tensor("bias", bias, (E, N), torch.float32, device)
    a.x_dtype = TORCH_TO_DTYPE[x.dtype].value
    a.input_dtype = DType.FP8.value if scaled else a.x_dtype
    a.x_stride_m, a.out_stride_m = (x.stride(0) if fits and rows > 1 else K), out_cols
    a.w_stride_e = (W_q.stride(0) if E > 1 else W_q.shape[1] * N) * W_q.element_size()
    if nbits == 4:
        a.meta_dtype = TORCH_TO_DTYPE[scales.dtype].value
        a.meta_stride_e = scales.stride(0) * 2
    elif nbits == 8:
        a.meta_dtype = DType.FP32.value
        a.meta_stride_e = scales.stride(0) * 4
    # (addresses that stand for the operands until the first launch sets them: checks look at alignment only)
    a.x = a.w = a.out = 4096
    a.scales = 4096 if scales.numel() > 0 else None
    a.zeros = 4096 if zeros.numel() > 0 and wgm != 2 else None
    return a, _ext.experts_workspace_need(a), (out_rows, out_cols), DTYPE_TO_TORCH[out_code]


def _launch(mode, x, bias, tensor_args, meta_args, offsets, plan, tile_config):
    W_q, scales, zeros = tensor_args[0], tensor_args[1], tensor_args[2]
    # whether the kernels can read the rows of x where they are (16-byte pieces); a copy is made of other ones
    fits = x.data_ptr() % 16 == 0 and x.dim() == 2 and x.stride(1) == 1 and (
        x.shape[0] <= 1 or (x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1]))
    key = (mode, fits, tile_config, _thread_id(), x.shape, x.stride(), x.dtype, x.device, W_q.shape, W_q.stride(), W_q.dtype, W_q.device,
           scales.shape, scales.stride(), scales.dtype, scales.device, zeros.shape, zeros.stride(), zeros.dtype, zeros.device,
           offsets.shape, offsets.stride(), offsets.dtype, offsets.device, *meta_args)
    if plan is not None:
        p = plan.order if mode == _GATED else plan.weights
        key += (plan.places.shape, plan.places.stride(), plan.places.dtype, plan.places.device, p.shape, p.stride(), p.dtype, p.device)
    if bias is not None:
        key += (bias.shape, bias.stride(), bias.dtype, bias.device)
    entry = _PREPARED.get(key)
    if entry is None:
        entry = _prepare(mode, x, fits, bias, tensor_args, meta_args, offsets, plan, tile_config)
        if len(_PREPARED) >= _PREPARED_LIMIT:
            _PREPARED.clear()
        _PREPARED[key] = entry
    a, need, out_shape, out_dtype = entry
    if not fits:
        x = x.clone(memory_format=torch.contiguous_format)
    out = x.new_empty(out_shape, dtype=out_dtype)
    a.x, a.w, a.out, a.offsets = x.data_ptr(), W_q.data_ptr(), out.data_ptr(), offsets.data_ptr()
    if a.scales is not None:
        a.scales = scales.data_ptr()
    if a.zeros is not None:
        a.zeros = zeros.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    if mode == _GATED:
        a.order = plan.order.data_ptr()
    elif mode == _COMBINED:
        a.places, a.weights = plan.places.data_ptr(), plan.weights.data_ptr()
    if out_shape[0] > 0:
        _ext.experts_matmul(a, need, x)
    return out


def experts_functional(x: Tensor, bias: Optional[Tensor], tensor_args: List[Tensor], meta_args: List[int], offsets: Tensor,
                       tile_config: int = -1) -> Tensor:
    """``out[r] = x[r] @ W[e(r)] (+ bias[e(r)])`` for rows [R, K] that are already grouped by expert: rows
    ``offsets[e] .. offsets[e + 1] - 1`` are expert ``e``'s, rows from ``offsets[E]`` on and in front of ``offsets[0]`` (above 0
    in a slice of longer offsets) come out as zeros.

    ``tensor_args = [W_q, scales, zeros]`` and ``meta_args`` are those of ``GemLiteLinear`` with a leading axis of experts
    on every tensor; ``bias`` is [E, N] fp32 and is added before the result is rounded.  fp8 experts quantise every row of
    ``x`` per 128 values: ``s = max(amax * fp32(1 / 448), 1e-6)``, ``code = e4m3(x * (1 / s))`` in fp32.  (The dense layers
    divide by 448 where this multiplies: a value on the border between two codes, which is where 16-bit values over
    their block's maximum often lie, may get the other neighbour.)
    """
    return _dispatch(_ROWS, x, bias, tensor_args, meta_args, offsets, None, tile_config)


def experts_gated_functional(x: Tensor, bias: Optional[Tensor], tensor_args: List[Tensor], meta_args: List[int], plan: ExpertPlan,
                             tile_config: int = -1) -> Tensor:
    """``silu(x[t] @ W_gate[e]) * (x[t] @ W_up[e])`` for every (token, expert) pair of the plan, as rows sorted by expert
    [T k, N / 2].  The first half of an expert's N columns is the gate, the second the up projection.  The activation is
    applied to the fp32 sums.  Rows without an expert are zeros."""
    return _dispatch(_GATED, x, bias, tensor_args, meta_args, plan.offsets, plan, tile_config)


def experts_combined_functional(h: Tensor, bias: Optional[Tensor], tensor_args: List[Tensor], meta_args: List[int], plan: ExpertPlan,
                                tile_config: int = -1) -> Tensor:
    """``sum over a token's slots of weight * (h[place] @ W[e])`` for rows ``h`` [T k, K] sorted by expert: [T, N].  Products
    and sum are fp32, rounded once; slots without an expert add nothing."""
    return _dispatch(_COMBINED, h, bias, tensor_args, meta_args, plan.offsets, plan, tile_config)


class GemLiteExperts(torch.nn.Module):
    """Packed ``GemLiteLinear`` layers of one kind, one per expert, in one set of tensors.

    Kinds: 4-bit codes in 32-bit words with group-wise or channel-wise scales (``A16W4_HQQ_INT``), fp8 with 128 x 128 block
    scales (``A8W8_fp8_dynamic(block_quant=True)``) and unquantised 16-bit weights (``W_nbits=16``).  The tensors are
    those of the layers with a leading axis of experts.
    """

    _SCHEMA = ("W_q", "scales", "zeros", "bias", "metadata")

    def __init__(self):
        super().__init__()
        for name in self._SCHEMA:
            self.register_buffer(name, None)
        self.meta_args = None

    @staticmethod
    def from_layers(layers) -> "GemLiteExperts":
        layers = list(layers)
        if not layers or not all(isinstance(layer, GemLiteLinear) for layer in layers):
            raise ValueError("from_layers takes a non-empty list of packed GemLiteLinear layers")
        first = layers[0]
        meta = first.get_meta_args()
        for i, layer in enumerate(layers):
            if layer.get_meta_args() != meta or layer.W_q.shape != first.W_q.shape or layer.scales.shape != first.scales.shape:
                raise ValueError(f"layer {i} is of another kind or shape than layer 0")
            if layer.W_q.device != first.W_q.device or layer.W_q.dtype != first.W_q.dtype or layer.scales.dtype != first.scales.dtype:
                raise ValueError(f"layer {i} has another device or type than layer 0")
            if (layer.bias is None) != (first.bias is None):
                raise ValueError(f"layer {i}: either all layers have a bias or none")
        nbits, e, csm, wgm = first.W_nbits, first.elements_per_sample, first.channel_scale_mode, first.W_group_mode
        K = first.in_features

        none = torch.empty(0, dtype=torch.int32, device=first.W_q.device)
        if nbits == 4 and e == 8 and not first.scaled_activations and first.W_q.dtype == torch.int32:
            if csm == 1 and wgm in (0, 1):  # one scale per channel, applied after the sum: the same product
                meta[2], meta[9], meta[10] = K, 0, 2 if wgm == 0 else 3
            elif csm != 0 or wgm not in (2, 3, 4):
                raise NotImplementedError(f"4-bit experts with W_group_mode {wgm} and channel_scale_mode {csm} are not built")
            if meta[2] % 32 != 0 or first.scales.dtype != DTYPE_TO_TORCH[first.output_dtype.value]:
                raise NotImplementedError(f"4-bit experts with groups of {meta[2]} and scales of type {first.scales.dtype} for outputs of type "
                                          f"{first.output_dtype} are not built")
            W_q = torch.stack([layer.W_q.data.contiguous() for layer in layers])
            scales = torch.stack([layer.scales.data.contiguous() for layer in layers])
            zeros = none
            if meta[10] != 2:
                zeros = torch.stack([GemLiteExperts._zeros_like_scales(layer) for layer in layers])
        elif nbits == 8 and e == 1 and csm == 5 and wgm == 0 and first.W_q.dtype == torch.float8_e4m3fn and first.scaled_activations:
            if K % 128 != 0:
                raise NotImplementedError(f"fp8 experts with K={K}: only multiples of 128 are built")
            # (moved as bytes: stacking is not implemented for every 8-bit float type)
            W_q = torch.stack([layer.W_q.data.t().contiguous().view(torch.uint8) for layer in layers])
            W_q = W_q.view(torch.float8_e4m3fn).transpose(1, 2)
            scales, zeros = torch.stack([layer.scales.data.contiguous() for layer in layers]), none
        elif nbits == 16 and e == 1 and csm == 0 and first.scales.numel() == 0 and first.W_q.dtype in (torch.float16, torch.bfloat16):
            if first.output_dtype != TORCH_TO_DTYPE[first.W_q.dtype]:
                raise NotImplementedError(f"16-bit experts of {first.W_q.dtype} with output type {first.output_dtype} are not built")
            meta[10] = 0
            W_q = torch.stack([layer.W_q.data.t().contiguous() for layer in layers]).transpose(1, 2)
            scales, zeros = none, none
        else:
            raise NotImplementedError(
                f"experts of layers with W_nbits={nbits}, {first.W_q.dtype} weights, W_group_mode={wgm} and channel_scale_mode={csm} are not "
                "built (4-bit codes in int32 words, fp8 with 128 x 128 block scales, 16-bit weights)")
        self = GemLiteExperts()
        bias = None if first.bias is None else torch.stack([layer.bias.data.float() for layer in layers]).contiguous()
        self._set(W_q, scales, zeros, bias, meta)
        return self

    @staticmethod
    def _zeros_like_scales(layer):
        z, s = layer.zeros.data, layer.scales.data
        if z.numel() == s.numel():
            if z.dtype != s.dtype:
                raise NotImplementedError(f"zeros of type {z.dtype} with scales of type {s.dtype} are not built")
            return z.reshape(s.shape).contiguous()
        if z.numel() != 1:
            raise NotImplementedError(f"zeros of shape {tuple(z.shape)} with scales of shape {tuple(s.shape)} are not built")
        full = z.reshape(1, 1).to(s.dtype).expand(s.shape).contiguous()
        if float(full.flatten()[0]) != float(z):
            raise NotImplementedError(f"a zero point of {float(z)} does not fit {s.dtype}")
        return full

    def _set(self, W_q, scales, zeros, bias, meta):
        self.W_q, self.scales, self.zeros, self.bias = W_q, scales, zeros, bias
        self.meta_args = [int(v) for v in meta]
        self.metadata = torch.tensor(self.meta_args, dtype=torch.int32, device=W_q.device)
        self.num_experts, self.out_features = W_q.shape[0], W_q.shape[2]
        self.in_features = W_q.shape[1] * self.meta_args[4]

    def get_tensor_args(self):
        return [self.W_q, self.scales, self.zeros]

    def get_meta_args(self):
        return list(self.meta_args)

    def forward(self, x: Tensor, offsets: Tensor) -> Tensor:
        """Rows already grouped by expert (``experts_functional``)."""
        return _dispatch(_ROWS, x, self.bias, self.get_tensor_args(), self.meta_args, offsets, None)

    def forward_gated(self, x: Tensor, plan: ExpertPlan) -> Tensor:
        """Gate and up projection of every (token, expert) pair (``experts_gated_functional``)."""
        return _dispatch(_GATED, x, self.bias, self.get_tensor_args(), self.meta_args, plan.offsets, plan)

    def forward_combined(self, h: Tensor, plan: ExpertPlan) -> Tensor:
        """Weighted sum of every token's experts (``experts_combined_functional``)."""
        return _dispatch(_COMBINED, h, self.bias, self.get_tensor_args(), self.meta_args, plan.offsets, plan)

    def extra_repr(self):
        if self.meta_args is None:
            return "empty"
        return f"experts={self.num_experts}, in_features={self.in_features}, out_features={self.out_features}, W_nbits={self.meta_args[1]}"

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        """Shapes and kind come from the checkpoint, as for ``GemLiteLinear``."""
        sd = {k: state_dict.pop(prefix + k, None) for k in self._SCHEMA}
        if sd["W_q"] is None or sd["metadata"] is None:
            missing_keys.extend(prefix + k for k in ("W_q", "metadata") if sd[k] is None)
            return
        try:
            meta = sd["metadata"].tolist()
            W_q = sd["W_q"]
            none = torch.empty(0, dtype=torch.int32, device=W_q.device)
            scales = none if sd["scales"] is None else sd["scales"]
            zeros = none if sd["zeros"] is None else sd["zeros"]
            if meta[1] >= 8 and W_q.stride(1) != 1:  # a checkpoint format that does not keep strides
                raw = W_q.view(torch.uint8) if W_q.dtype == torch.float8_e4m3fn else W_q
                W_q = raw.transpose(1, 2).contiguous().view(W_q.dtype).transpose(1, 2)
            _weights_of([W_q, scales, zeros], meta)
            self._set(W_q, scales, zeros, sd["bias"], meta)
        except Exception as exc:  # reported through nn.Module's error list
            error_msgs.append(f"GemLiteExperts load error at prefix '{prefix}': {exc}")


class GemLiteMoE(torch.nn.Module):
    """Router, gated projection and combined projection of a mixture-of-experts block.

    ``gate_up``: experts with the gate columns followed by the up columns; ``down``: experts back to the model's width.
    ``forward(x, logits)``: x [..., hidden], router logits [..., experts].  Two empty ``GemLiteExperts`` make a block that
    ``load_state_dict`` fills.
    """

    def __init__(self, gate_up: GemLiteExperts, down: GemLiteExperts, top_k: int, scoring: str = "softmax", renormalize: bool = True,
                 scale: float = 1.0):
        super().__init__()
        if scoring not in SCORINGS:
            raise ValueError(f"scoring: expected one of {sorted(SCORINGS)}, got {scoring!r}")
        self.gate_up, self.down = gate_up, down
        self.top_k, self.scoring, self.renormalize, self.scale = top_k, scoring, renormalize, scale
        if gate_up.meta_args is not None or down.meta_args is not None:
            self._check_pair()

    def _check_pair(self):
        up, down = self.gate_up, self.down
        if up.meta_args is None or down.meta_args is None or up.num_experts != down.num_experts or up.out_features != 2 * down.in_features:
            raise ValueError(f"gate_up ({up.extra_repr()}) and down ({down.extra_repr()}) do not belong together")

    def forward(self, x: Tensor, logits: Tensor) -> Tensor:
        self._check_pair()
        x2d, logits2d = x.reshape(-1, x.shape[-1]), logits.reshape(-1, logits.shape[-1])
        if x2d.shape[0] != logits2d.shape[0] or logits2d.shape[1] != self.gate_up.num_experts:
            raise ValueError(f"x of shape {tuple(x.shape)} and logits of shape {tuple(logits.shape)} for {self.gate_up.num_experts} experts")
        plan = route_experts(logits2d, self.top_k, self.scoring, self.renormalize, self.scale)
        y = self.down.forward_combined(self.gate_up.forward_gated(x2d, plan), plan)
        return y.view(x.shape[:-1] + (self.down.out_features,))


# ---------------------------------------------------------------------------
# the same calls as custom ops, so that torch.compile holds each as one node (eager calls do not pay the op dispatch)
# ---------------------------------------------------------------------------
def _make_custom_ops():
    try:
        @torch.library.custom_op("gemlite::route_experts", mutates_args=())
        def route_experts_op(logits: Tensor, top_k: int, scoring: str, renormalize: bool, scale: float) -> List[Tensor]:
            # (the outputs of an op must not share memory)
            return list(_route_experts(logits, top_k, scoring, renormalize, scale, apart=True))

        @route_experts_op.register_fake
        def _(logits, top_k, scoring, renormalize, scale):
            T, E = logits.shape
            ints = dict(dtype=torch.int32, device=logits.device)
            return [torch.empty((T, top_k), dtype=torch.float32, device=logits.device), torch.empty((T, top_k), **ints),
                    torch.empty((E + 1,), **ints), torch.empty((T * top_k,), **ints), torch.empty((T, top_k), **ints)]

        @torch.library.custom_op("gemlite::experts", mutates_args=())
        def experts_op(mode: int, x: Tensor, bias: Optional[Tensor], tensor_args: List[Tensor], meta_args: List[int], offsets: Tensor,
                       plan: List[Tensor], tile_config: int = -1) -> Tensor:
            return _launch(mode, x, bias, tensor_args, meta_args, offsets, ExpertPlan(*plan) if plan else None, tile_config)

        @experts_op.register_fake
        def _(mode, x, bias, tensor_args, meta_args, offsets, plan, tile_config=-1):
            N, rows = tensor_args[0].shape[2], x.shape[0]
            if mode != _ROWS:
                T, k = plan[4].shape
                rows = T if mode == _COMBINED else T * k
            return torch.empty((rows, N // 2 if mode == _GATED else N), dtype=DTYPE_TO_TORCH[int(meta_args[6])], device=x.device)

        return route_experts_op, experts_op
    except Exception as exc:  # a name is taken or torch is too old
        logger.warning("gemlite_amd: torch custom ops gemlite::route_experts and gemlite::experts were not registered (%s); "
                       "torch.compile will trace into the plain Python calls", exc)
        return None, None


route_experts_op, experts_op = _make_custom_ops()


def _dispatch(mode, x, bias, tensor_args, meta_args, offsets, plan, tile_config=-1):
    if experts_op is not None and torch.compiler.is_compiling():
        return experts_op(mode, x, bias, tensor_args, meta_args, offsets, [] if plan is None else list(plan), tile_config)
    return _launch(mode, x, bias, tensor_args, meta_args, offsets, plan, tile_config)


__all__ = [
    "ExpertPlan",
    "GemLiteExperts",
    "GemLiteMoE",
    "experts_combined_functional",
    "experts_functional",
    "experts_gated_functional",
    "plan_experts",
    "route_experts",
]
