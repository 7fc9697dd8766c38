"""IMA_STUDENT_KERNEL plugin surface on B200 (drop-in for the student side of the
reference's __main__.py).

Same module-level configuration (env vars read at import, __main__.py:39-50), the
same student modules (CodebookLinear, HawkeyeLinear, HawkeyeClassCountsLinear and
the non-FP8 Int32Linear, __main__.py:390-523), the same kernel wrappers
(_int32_raw_matmul :228-253, _int32_matmul :301-333), the same probe
(_Int32KernelProbe :667-678, bumped once per checkable integer product) and the
same replacement pass (_replace_int32_linears :563-588).  One kernel more: "int8",
plain 8-bit linears and gated blocks (Int8Linear, Int8GatedMLP).  Every integer product
runs on the sm_100a kernels of libima_b200.so; there is no CPU execution path.
"""

from __future__ import annotations

import copy
import functools
import inspect
import math
import os
from typing import Any

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _native as nat
from .codebook import DigitPlanes, codebook_planes_from_fp8, int_gemm, per_token_fp8, planes_from_int32
from .hawkeye import _validate_params as _validate_hawkeye_params
from .hawkeye import hawkeye_replay, quantize_and_stage, stage_weight
from .hawkeye_freivalds import exact_hawkeye_fp8_sum, stage_class_count_weight
from .int8 import ACTIVATIONS as INT8_ACTIVATIONS
from .int8 import Int8Weight, int8_gated, int8_linear

STUDENT_KERNEL = os.environ.get("IMA_STUDENT_KERNEL", "codebook")
# "int8" (no counterpart in the reference): every linear as an Int8Linear, gated blocks fused
SUPPORTED_STUDENT_KERNELS = {"codebook", "hawkeye", "hawkeye-class-counts", "int8"}
HAWKEYE_PRODUCTS_PER_GROUP = int(os.environ.get("IMA_HAWKEYE_GROUP", "32"))
HAWKEYE_INTERNAL_WIDTH = int(os.environ.get("IMA_HAWKEYE_WIDTH", "14"))
HAWKEYE_CLASS_CHUNK = int(os.environ.get("IMA_HAWKEYE_CLASS_CHUNK", "32"))
HAWKEYE_PACKED_COUNT_LANES = int(os.environ.get("IMA_HAWKEYE_PACKED_COUNT_LANES", "6"))
HAWKEYE_PACKED_GROUP_LANES = int(os.environ.get("IMA_HAWKEYE_PACKED_GROUP_LANES", "1"))
HAWKEYE_ZERO_EXPONENT = -139
HAWKEYE_BLOCK_M = int(os.environ.get("IMA_HAWKEYE_BLOCK_M", "4"))
HAWKEYE_BLOCK_N = int(os.environ.get("IMA_HAWKEYE_BLOCK_N", "32"))

FP8_E4M3_MAX = 448.0
FP8_E4M3_CODE_SCALE = 512.0
INT32_MAX = (1 << 31) - 1
INT64_ACCUM_LIMIT = (1 << 62) - 1
_ACTIVE_INT32_PROBE = None

_PLANES_ATTR = "_ima_planes"


def _require_cuda_tensor(x: torch.Tensor, label: str) -> None:
    if x.device.type != "cuda":
        raise RuntimeError(f"{label} must be on CUDA; this repo has no CPU execution path")


_version_of = nat.tensor_version


def _attach_planes(t: torch.Tensor, planes: DigitPlanes) -> None:
    """Remember the digit planes of an int32 operand on the tensor object itself, so that
    _int32_matmul can skip re-expanding it.  The planes are used only while the tensor's
    version counter is unchanged, so an in-place edit invalidates them.  Inference tensors
    have no version counter: nothing is cached for them (this package creates its own
    int32 operands as normal tensors, even inside inference mode, so they stay cacheable)."""
    version = _version_of(t)
    if version is None:
        return
    try:
        setattr(t, _PLANES_ATTR, (planes, version, t.data_ptr()))
    except (AttributeError, RuntimeError):
        pass


def _attached_planes(t: torch.Tensor) -> DigitPlanes | None:
    entry = getattr(t, _PLANES_ATTR, None)
    if entry is None:
        return None
    planes, version, data_ptr = entry
    current = _version_of(t)
    if current is None or current != version or t.data_ptr() != data_ptr:
        return None
    return planes


def _owned_copy(weight: torch.Tensor) -> torch.Tensor:
    """A module-owned contiguous copy of an FP8 weight, created as a normal (versioned)
    tensor even inside inference mode, so that the staging cached on it is dropped after
    an in-place edit."""
    with torch.inference_mode(False):
        return weight.detach().clone(memory_format=torch.contiguous_format)


# ---------------------------------------------------------------------------
# quantisers (ref __main__.py:148-185)
# ---------------------------------------------------------------------------
def _per_token_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda_tensor(x, "FP8 activation")
    q, scale, _cb, _cs, _dp = per_token_fp8(x)
    return q, scale


def _fp8_e4m3_to_int32(x: torch.Tensor) -> torch.Tensor:
    _require_cuda_tensor(x, "FP8 codebook source")
    raw = x.contiguous().view(torch.uint8)
    shape = raw.shape
    rows = raw.reshape(-1, shape[-1]) if raw.ndim > 1 else raw.reshape(1, -1)
    out = torch.empty(rows.shape, dtype=torch.int32, device=raw.device)
    with torch.cuda.device(raw.device):
        nat.call(
            "ima_codebook_from_fp8", rows.data_ptr(), rows.shape[0], rows.shape[1], rows.shape[1], out.data_ptr(),
            rows.shape[1], nat.stream_of(raw.device),
        )
    return out.reshape(shape)


def _per_token_fp8_int32(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda_tensor(x, "FP8 activation")
    _q, _scale, codebook, code_scale, planes = per_token_fp8(x, codebook=True, planes=True)
    _attach_planes(codebook, planes)
    return codebook, code_scale


def _int32_qmax(k: int) -> float:
    # Keep worst-case sum_k(qmax*qmax) inside signed int64 with headroom.
    return float(min(INT32_MAX, int(math.sqrt(INT64_ACCUM_LIMIT / max(k, 1)))))


def _per_token_int32(x: torch.Tensor, qmax: float) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda_tensor(x, "int32 activation")
    rows = x.reshape(-1, x.shape[-1])
    scale = rows.detach().abs().amax(dim=-1, keepdim=True).to(torch.float32)
    scale = (scale / qmax).clamp_min(1e-12)
    q = (rows.to(torch.float32) / scale).round().clamp(-qmax, qmax)
    return q.to(torch.int32).contiguous(), scale


def _per_row_int32(weight: torch.Tensor, qmax: float) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda_tensor(weight, "int32 weight source")
    w = weight.detach().to(torch.float32)
    scale = (w.abs().amax(dim=1, keepdim=True) / qmax).clamp_min(1e-12)
    q = (w / scale).round().clamp(-qmax, qmax)
    return q.to(torch.int32).contiguous(), scale.to(torch.float32)


# ---------------------------------------------------------------------------
# integer GEMM wrappers (ref __main__.py:228-333)
# ---------------------------------------------------------------------------
def _operand_planes(activations: torch.Tensor, weight_t: torch.Tensor) -> tuple[DigitPlanes, DigitPlanes]:
    a = _attached_planes(activations)
    b = _attached_planes(weight_t)
    if a is not None and b is not None and a.scheme == b.scheme:
        return a, b
    # Unknown int32 values: the five-digit scheme is exact for every int32.
    if a is None or a.scheme != nat.IMA_SCHEME_DIGITS5:
        a = planes_from_int32(activations, scheme=nat.IMA_SCHEME_DIGITS5)
    if b is None or b.scheme != nat.IMA_SCHEME_DIGITS5:
        b = planes_from_int32(weight_t, transpose=True, scheme=nat.IMA_SCHEME_DIGITS5)
    return a, b


def _int32_raw_matmul(activations: torch.Tensor, weight_t: torch.Tensor) -> torch.Tensor:
    global _ACTIVE_INT32_PROBE
    _require_cuda_tensor(activations, "int32 activation matrix")
    _require_cuda_tensor(weight_t, "int32 weight matrix")
    if activations.dtype != torch.int32 or weight_t.dtype != torch.int32:
        raise RuntimeError("int32 raw matmul received non-int32 operands")
    m_size, k_size = activations.shape
    k2, n_size = weight_t.shape
    if k_size != k2:
        raise RuntimeError(f"int32 raw matmul shape mismatch: {activations.shape} @ {weight_t.shape}")
    out = torch.empty((m_size, n_size), device=activations.device, dtype=torch.int64)
    if _ACTIVE_INT32_PROBE is not None:
        _ACTIVE_INT32_PROBE.count += 1
    a, b = _operand_planes(activations, weight_t)
    int_gemm(a, b, c_out=out)
    return out


def _int32_matmul(
    activations: torch.Tensor,
    weight_t: torch.Tensor,
    x_scale: torch.Tensor,
    w_scale: torch.Tensor,
) -> torch.Tensor:
    global _ACTIVE_INT32_PROBE
    _require_cuda_tensor(activations, "int32 activation matrix")
    _require_cuda_tensor(weight_t, "int32 weight matrix")
    if activations.dtype != torch.int32 or weight_t.dtype != torch.int32:
        raise RuntimeError("int32 matmul received non-int32 operands")
    m_size, k_size = activations.shape
    k2, n_size = weight_t.shape
    if k_size != k2:
        raise RuntimeError(f"int32 matmul shape mismatch: {activations.shape} @ {weight_t.shape}")
    out = torch.empty((m_size, n_size), device=activations.device, dtype=torch.float32)
    if _ACTIVE_INT32_PROBE is not None:
        _ACTIVE_INT32_PROBE.count += 1
    a, b = _operand_planes(activations, weight_t)
    int_gemm(a, b, want_c=False, x_scale=x_scale, w_scale=w_scale, y_out=out)
    return out


# ---------------------------------------------------------------------------
# student modules (ref __main__.py:390-523)
# ---------------------------------------------------------------------------
class Int32Linear(nn.Module):
    """Linear backed by the exact int32 tensor-core GEMM (non-FP8 linears)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None):
        super().__init__()
        _require_cuda_tensor(weight, "int32 weight source")
        self.qmax = _int32_qmax(weight.shape[1])
        w_i32, w_scale = _per_row_int32(weight, self.qmax)
        self.register_buffer("weight_t", w_i32.t().contiguous(), persistent=False)
        self.register_buffer("weight_scale", w_scale.reshape(1, -1), persistent=False)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach(), persistent=False)
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _require_cuda_tensor(x, "int32 input")
        in_shape = x.shape
        x_i32, x_scale = _per_token_int32(x, self.qmax)
        y = _int32_matmul(x_i32, self.weight_t, x_scale, self.weight_scale)
        if self.bias is not None:
            y = y + self.bias.to(torch.float32)
        return y.to(x.dtype).reshape(*in_shape[:-1], self.out_features)


class CodebookLinear(nn.Module):
    """FP8 linear reconstructed by one Freivalds-checkable codebook integer GEMM."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None):
        super().__init__()
        if weight.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"CodebookLinear needs FP8 weights, got {weight.dtype}")
        _require_cuda_tensor(weight, "FP8 codebook weight")
        planes, codebook_t = codebook_planes_from_fp8(weight.detach(), with_codebook_t=True)
        codebook_scale = weight_scale.detach().to(torch.float32) / FP8_E4M3_CODE_SCALE
        self.register_buffer("weight_t", codebook_t, persistent=False)
        self.register_buffer("weight_scale", codebook_scale.reshape(1, -1), persistent=False)
        _attach_planes(self.weight_t, planes)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach(), persistent=False)
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _require_cuda_tensor(x, "FP8 codebook input")
        in_shape = x.shape
        x_i32, x_scale = _per_token_fp8_int32(x)
        y = _int32_matmul(x_i32, self.weight_t, x_scale, self.weight_scale)
        if self.bias is not None:
            y = y + self.bias.to(torch.float32)
        return y.to(x.dtype).reshape(*in_shape[:-1], self.out_features)


class HawkeyeLinear(nn.Module):
    """FP8 linear reconstructed by direct Hawkeye integer replay."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None):
        super().__init__()
        if weight.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"HawkeyeLinear needs FP8 weights, got {weight.dtype}")
        _require_cuda_tensor(weight, "Hawkeye FP8 weight")
        self.register_buffer("weight", _owned_copy(weight), persistent=False)
        self.register_buffer("weight_scale", weight_scale.detach().to(torch.float32), persistent=False)
        stage_weight(self.weight)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach(), persistent=False)
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _require_cuda_tensor(x, "Hawkeye input")
        in_shape = x.shape
        # the reference's _fp8_per_token then hawkeye_fp8_sum (__main__.py:467-481), with the
        # quantisation and the activation staging fused into one launch, then the replay;
        # the replay parameters are validated as hawkeye_fp8_sum validates them
        _validate_hawkeye_params(HAWKEYE_PRODUCTS_PER_GROUP, HAWKEYE_INTERNAL_WIDTH, HAWKEYE_ZERO_EXPONENT)
        x_op, x_scale, _ = quantize_and_stage(x)
        y = hawkeye_replay(x_op, stage_weight(self.weight), x_scale, self.weight_scale)
        if self.bias is not None:
            y = y + self.bias.to(y.dtype)
        return y.to(x.dtype).reshape(*in_shape[:-1], self.out_features)


class HawkeyeClassCountsLinear(nn.Module):
    """FP8 linear reconstructed exactly from checkable Hawkeye class-count products."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None):
        super().__init__()
        if weight.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"HawkeyeClassCountsLinear needs FP8 weights, got {weight.dtype}")
        _require_cuda_tensor(weight, "Hawkeye exact FP8 weight")
        self.register_buffer("weight", _owned_copy(weight), persistent=False)
        self.register_buffer("weight_scale", weight_scale.detach().to(torch.float32), persistent=False)
        stage_class_count_weight(self.weight)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach(), persistent=False)
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _require_cuda_tensor(x, "Hawkeye exact input")
        in_shape = x.shape
        x_fp8, x_scale = _per_token_fp8(x)
        # raw_matmul None: the class-count engine forms the checkable count products on the
        # tensor cores (the reference passes its _int32_raw_matmul here, which forms them)
        y, _stats = exact_hawkeye_fp8_sum(
            x_fp8,
            x_scale,
            self.weight,
            self.weight_scale,
            None,
            products_per_group=HAWKEYE_PRODUCTS_PER_GROUP,
            internal_width=HAWKEYE_INTERNAL_WIDTH,
            zero_exponent=HAWKEYE_ZERO_EXPONENT,
            class_chunk=HAWKEYE_CLASS_CHUNK,
            packed_count_lanes=HAWKEYE_PACKED_COUNT_LANES,
            packed_group_lanes=HAWKEYE_PACKED_GROUP_LANES,
        )
        if self.bias is not None:
            y = y + self.bias.to(y.dtype)
        return y.to(x.dtype).reshape(*in_shape[:-1], self.out_features)


class Int8Linear(nn.Module):
    """Linear with int8 activations (one scale per token) and int8 weights (one per output channel):
    one exact int32 product per forward, counted by the probe.  No counterpart in the reference.  Made from
    the dequantised weight, like Int32Linear; the buffers weight and weight_scale hold its codes and scales."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None):
        super().__init__()
        _require_cuda_tensor(weight, "int8 weight source")
        with torch.inference_mode(False):   # versioned even inside inference mode (see _owned_copy)
            handle = Int8Weight.from_float(weight.detach())
        self._handle = handle
        self.register_buffer("weight", handle.codes, persistent=False)
        self.register_buffer("weight_scale", handle.scale, persistent=False)
        if bias is None:
            self.bias = None
        else:
            self.register_buffer("bias", bias.detach(), persistent=False)
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0]

    def _apply(self, fn, recurse=True):
        """The module moved (model.to and the like).  The scales belong to the codes: a cast of the model's floating
        tensors leaves them in fp32."""
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def int8_weight(self) -> Int8Weight:
        """The codes and scales as int8_linear takes them (laid out anew if a buffer was replaced,
        e.g. by moving the module)."""
        if self._handle.codes is not self.weight or self._handle.scale is not self.weight_scale:
            self._handle = Int8Weight(self.weight, self.weight_scale)
            self.weight, self.weight_scale = self._handle.codes, self._handle.scale
        return self._handle

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _require_cuda_tensor(x, "int8 input")
        _bump_probe(1)
        return int8_linear(x, self.int8_weight(), self.bias)


class Int8GatedMLP(nn.Module):
    """Gated feed-forward block down(act(gate(x)) * up(x)) on three Int8Linear: gate, up, activation and
    product in one kernel, then the down projection.  While gate_proj or up_proj has a hook, both are
    called as modules and their outputs rounded to x's type."""

    def __init__(self, gate_proj: Int8Linear, up_proj: Int8Linear, down_proj: Int8Linear, activation: str):
        super().__init__()
        if activation not in INT8_ACTIVATIONS:
            raise RuntimeError(f"unknown activation {activation!r}; choose one of: {', '.join(sorted(INT8_ACTIVATIONS))}")
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if _hooked(self.gate_proj) or _hooked(self.up_proj):
            return self.down_proj(_ACTIVATION_FUNCTIONS[self.activation](self.gate_proj(x)) * self.up_proj(x))
        _require_cuda_tensor(x, "int8 input")
        _bump_probe(2)
        h = int8_gated(x, self.gate_proj.int8_weight(), self.up_proj.int8_weight(), self.gate_proj.bias,
                       self.up_proj.bias, activation=self.activation)
        return self.down_proj(h)


def _bump_probe(products: int) -> None:
    if _ACTIVE_INT32_PROBE is not None:
        _ACTIVE_INT32_PROBE.count += products


def _gated_activation(module: nn.Module) -> str | None:
    """The activation of a module that computes down(act(gate(x)) * up(x)) on children gate_proj, up_proj, down_proj
    and act_fn, in the layout of every gated block this package's shapes come from; None for anything else.
    The names only propose: a fused block replaces the module's own forward and no longer calls gate_proj, up_proj
    and act_fn, so own parameters or buffers (the activation's too), hooks on any of them and a forward that computes
    something else decline.  The activation may be of any class."""
    children = dict(module.named_children())
    if set(children) != {"gate_proj", "up_proj", "down_proj", "act_fn"}:
        return None
    act = children["act_fn"]
    own = (*module.parameters(recurse=False), *module.buffers(recurse=False), *act.parameters(), *act.buffers())
    if own or any(map(_hooked, (module, children["gate_proj"], children["up_proj"], *act.modules()))):
        return None
    return next((name for name in _ACTIVATION_FUNCTIONS if _computes_gated(module, name)), None)


_ACTIVATION_FUNCTIONS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": functools.partial(F.gelu, approximate="tanh")}


def _hooked(module: nn.Module) -> bool:
    return any(getattr(module, hooks, None) for hooks in (
        "_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks"))


class _Picked(nn.Module):
    """Stand-in for a projection: every output is one of the inputs times a factor."""

    def __init__(self, linear: nn.Module, step: int):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        i = torch.arange(self.out_features, device="cpu", dtype=torch.float64)
        self.index, self.factor = (step * (i + 1)).long() % self.in_features, 0.5 + (0.618 * step * (i + 1)) % 1.0

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x[..., self.index] * self.factor


def _computes_gated(module: nn.Module, activation: str) -> bool:
    """Whether module.forward(x) is down(act(gate(x)) * up(x)): run on the host in 64 bits with stand-ins for the
    three projections, on values of both signs from 1e-3 to 1e4, in training and in evaluation mode."""
    try:
        if "forward" in vars(module) or len(inspect.signature(module.forward).parameters) != 1:
            return False
        gate, up, down = (_Picked(getattr(module, name), step)
                          for name, step in (("gate_proj", 7), ("up_proj", 11), ("down_proj", 13)))
        tokens = max(3, -(-4096 // gate.in_features))   # narrow blocks too see every magnitude
        i = torch.arange(2 * tokens * gate.in_features, device="cpu", dtype=torch.float64).reshape(2, tokens, -1)
        x = torch.where(i * 0.7548 % 1.0 < 0.5, -1.0, 1.0) * 10.0 ** (7.0 * (i * 0.5698 % 1.0) - 3.0)
        want = down(_ACTIVATION_FUNCTIONS[activation](gate(x)) * up(x))
        bound = 1e-5 * want.abs() + down(1e-6 * up(x).abs())   # covers an activation taken in fp32
        for training in (False, True):
            twin = object.__new__(type(module))   # the module's own forward and attributes, other projections
            vars(twin).update(vars(module), training=training, _modules={
                "gate_proj": gate, "up_proj": up, "down_proj": down, "act_fn": copy.deepcopy(module.act_fn).train(training)})
            with torch.no_grad(), torch.random.fork_rng(devices=[]):
                got = twin.forward(x.clone())
            if not (isinstance(got, torch.Tensor) and got.shape == want.shape and
                    bool(((got.double() - want).abs() <= bound).all())):
                return False
    except Exception:   # a forward that needs more than its projections' outputs is not this formula
        return False
    return True


def _fuse_gated_blocks(model: nn.Module) -> None:
    """Replace every gated block (_gated_activation) whose three projections are Int8Linear by an Int8GatedMLP."""
    blocks = [(name, module) for name, module in model.named_modules() if name]
    for name, module in blocks:
        activation = _gated_activation(module)
        if activation is None:
            continue
        parts = [module.gate_proj, module.up_proj, module.down_proj]
        if all(isinstance(p, Int8Linear) for p in parts) and parts[0].weight.shape == parts[1].weight.shape:
            _set_submodule(model, name, Int8GatedMLP(*parts, activation))


# ---------------------------------------------------------------------------
# model integerisation (ref __main__.py:526-594)
# ---------------------------------------------------------------------------
def _expanded_block_scale(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    if scale.shape == weight.shape:
        return scale
    row_block = math.ceil(weight.shape[0] / scale.shape[0])
    col_block = math.ceil(weight.shape[1] / scale.shape[1])
    return scale.repeat_interleave(row_block, 0).repeat_interleave(col_block, 1)[
        : weight.shape[0], : weight.shape[1]
    ]


def _channel_scale(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """weight_scale of an FP8 linear as a factor of weight [N, K]: one scale, or one per output channel in any
    shape of N entries, as CodebookLinear reads it."""
    if scale.numel() not in (1, weight.shape[0]):
        raise RuntimeError(f"FP8 weight_scale has shape {tuple(scale.shape)}, expected one entry or one per output channel "
                           f"({weight.shape[0]})")
    return scale.to(torch.float32).reshape(-1, 1)


def _dequantized_weight(module: nn.Linear) -> torch.Tensor:
    weight = module.weight.detach()
    if weight.dtype == torch.float8_e4m3fn:
        if hasattr(module, "weight_scale"):
            return weight.to(torch.float32) * _channel_scale(weight, module.weight_scale.detach())
        if hasattr(module, "weight_scale_inv"):
            scale = module.weight_scale_inv.detach().to(torch.float32)
            return weight.to(torch.float32) * _expanded_block_scale(weight, scale)
        raise RuntimeError("FP8 Linear is missing a recognized weight scale")
    return weight.to(torch.float32)


def _replace_int32_linears(model: nn.Module) -> list[str]:
    if STUDENT_KERNEL not in SUPPORTED_STUDENT_KERNELS:
        supported = ", ".join(sorted(SUPPORTED_STUDENT_KERNELS))
        raise RuntimeError(f"unknown IMA_STUDENT_KERNEL={STUDENT_KERNEL!r}; choose one of: {supported}")
    replacements: list[tuple[str, nn.Linear]] = []
    for name, module in model.named_modules():
        if isinstance(module, nn.Linear):
            replacements.append((name, module))
    for name, module in replacements:
        if STUDENT_KERNEL == "int8":
            replacement = Int8Linear(_dequantized_weight(module), module.bias)
        elif module.weight.dtype == torch.float8_e4m3fn and hasattr(module, "weight_scale"):
            if STUDENT_KERNEL == "hawkeye":
                replacement = HawkeyeLinear(module.weight, module.weight_scale, module.bias)
            elif STUDENT_KERNEL == "hawkeye-class-counts":
                replacement = HawkeyeClassCountsLinear(module.weight, module.weight_scale, module.bias)
            else:
                replacement = CodebookLinear(module.weight, module.weight_scale, module.bias)
        else:
            replacement = Int32Linear(_dequantized_weight(module), module.bias)
        _set_submodule(model, name, replacement)
    if not replacements:
        raise RuntimeError("No Linear modules were found to integerize.")
    if STUDENT_KERNEL == "int8":
        _fuse_gated_blocks(model)
    return [name for name, _ in replacements]


def _set_submodule(model: nn.Module, name: str, replacement: nn.Module) -> None:
    parent_name, _, child_name = name.rpartition(".")
    parent = model.get_submodule(parent_name) if parent_name else model
    setattr(parent, child_name, replacement)


class _Int32KernelProbe:
    def __init__(self):
        self.count = 0

    def __enter__(self) -> "_Int32KernelProbe":
        global _ACTIVE_INT32_PROBE
        _ACTIVE_INT32_PROBE = self
        return self

    def __exit__(self, exc_type: Any, exc: Any, tb: Any) -> None:
        global _ACTIVE_INT32_PROBE
        _ACTIVE_INT32_PROBE = None
