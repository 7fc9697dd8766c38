"""8-bit integer linears (W8A8): one int8 scale per token and per output channel.

The codebook student reproduces an FP8 linear bit for bit and pays nine int8 products per
multiplication for it.  The operators here pay one: activations are quantised per token and
weights per output channel to int8, the product is exact in int32, and the scales are applied in
the epilogue.  int8_gemm returns the int32 product, which Freivalds checks like every integer
product of this package; int8_linear and int8_gated keep theirs on the chip.
There is no counterpart in the reference.

  per_token_int8    the quantiser of both sides
  Int8Weight        a weight's codes and channel scales, laid out once
  int8_gemm         codes in, exact int32 product and/or rescaled output (beside codebook.int_gemm)
  int8_linear       y = x W^T + b
  int8_gated        h = act(x Wg^T + bg) * (x Wu^T + bu), both projections, activation and product
                    in one kernel
  int8_linear_backward, int8_gated_backward   their gradients as plain calls

int8_linear and int8_gated take part in reverse-mode autograd; forward-mode tangents are refused.  A
whole training step can be captured into a CUDA graph if no eager autograd graph of the same leaves
is alive (refused where these operators recorded it; nothing tells of one that others recorded); the
*_backward calls, which record nothing, can always.
Gradients pass straight through the rounding: they are the derivatives at the dequantised
activations and weights, with the scales held fixed.  A weight given as a floating tensor is quantised in the call and gets a
gradient (training with a master weight); an Int8Weight is frozen and gets none.  The two
products of a backward pass run on the int8 tensor cores too: the gradient is written in
base-256 digits of its row maximum (two digits for bf16 tensors and sums of up to 65,536, else three;
see csrc/int8_quant.cu).

Shapes: every contraction (K; in the backward pass also the padded pair of N for the gated block, and
the number of tokens for a weight gradient) is at most 131071, so that int32 sums are exact.  N of a
linear is not limited: the activations' gradient of a wider one (a vocabulary head) is summed in fp32
from parts, of at most 65,536 outputs where two digits are taken.  Rows whose activations hold a NaN
or an infinity come out as NaN, as do rows of a product with a gradient that does.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat

MAX_K = 131071
TWO_DIGITS = 1 << 16   # longest sum that two digits of a bf16 gradient do for (_digit_count)
ACTIVATIONS = {"silu": nat.IMA_ACT_SILU, "gelu": nat.IMA_ACT_GELU, "gelu_tanh": nat.IMA_ACT_GELU_TANH}


_DTYPE_CODES = {torch.float32: nat.IMA_DTYPE_F32, torch.bfloat16: nat.IMA_DTYPE_BF16, torch.float16: nat.IMA_DTYPE_F16}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(dev: torch.device, fn: str, *args) -> None:
    """A C entry whose last argument is the stream, on `dev` and its current stream."""
    index = dev.index
    if _current_device() == index:
        status = getattr(nat.lib(), fn)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            status = getattr(nat.lib(), fn)(*args, _raw_stream(index))
    if status:
        raise nat.NativeError(fn, status)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _round_up(v: int, to: int) -> int:
    return (v + to - 1) // to * to


def _require_cuda(t: torch.Tensor, label: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{label} must be on CUDA; this repo has no CPU execution path")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t [..., K] as a matrix whose rows are contiguous and do not overlap (a copy if need be)."""
    r = t if t.ndim == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    (ld, step), (m, k) = r.stride(), r.shape
    if (step != 1 and k > 1) or (m > 1 and ld < k):
        r = r.contiguous()
    return r


def _ld(t: torch.Tensor) -> int:
    """Row stride of a matrix from _rows (a single row has none of its own)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _empty_codes(rows: int, k: int, like: torch.Tensor) -> torch.Tensor:
    """int8 [rows, k] whose rows start on 16 bytes, on the device of `like`."""
    ld = _round_up(max(k, 1), 16)
    t = like.new_empty((rows, ld), dtype=torch.int8)
    return t if ld == k else t[:, :k]


def _check_codes(t: torch.Tensor, label: str) -> None:
    if t.dtype is not torch.int8 or t.ndim != 2:
        raise RuntimeError(f"{label} must be a 2-D int8 tensor, got {t.dtype} {tuple(t.shape)}")
    if not t.is_cuda:
        _require_cuda(t, label)
    if t.shape[1] > MAX_K:
        raise RuntimeError(f"{label}: contraction of {t.shape[1]} exceeds {MAX_K} (exact int32 sums)")


def _layout(t: torch.Tensor, rows: int, k: int) -> tuple[int, int] | None:
    """(address, row stride) of an int8 matrix that the kernels can load, None if it has to be moved first."""
    at, (ld, step) = t.data_ptr(), t.stride()
    if rows <= 1 or k == 0:
        ld = _round_up(max(k, 1), 16)
    elif ld % 16 or ld < k:
        return None
    if at % 16 or step != 1 and k > 1:
        return None if rows and k else (at, ld)
    return at, ld


def _aligned_codes(t: torch.Tensor, label: str) -> torch.Tensor:
    """An int8 matrix as the kernels load it: contiguous rows that start on 16 bytes (a copy
    only if it is not)."""
    _check_codes(t, label)
    return t if _layout(t, *t.shape) else _packed_codes(t)[0]


def _packed_codes(*given: torch.Tensor) -> list[torch.Tensor]:
    """Copies of one or two int8 matrices of one width and device, in rows that start on 16 bytes; one
    launch where their columns are contiguous."""
    k = given[0].shape[1]
    out = [_empty_codes(t.shape[0], k, t) for t in given]
    args = []
    for t, o in zip(given, out):
        if (t.stride(1) == 1 or k == 1) and (t.shape[0] <= 1 or t.stride(0) >= k):
            args += [t.data_ptr(), t.shape[0], _ld(t), o.data_ptr()]
        elif t.stride(0) == 1 and t.stride(1) >= t.shape[0]:
            _call(t.device, "ima_int8_transpose", t.data_ptr(), k, t.shape[0], t.stride(1), o.data_ptr(), _code_ld(o))
        else:
            o.copy_(t)
    if args:
        args += [None, 0, 0, None] if len(args) == 4 else []
        _call(out[0].device, "ima_int8_pack_rows", *args, k, _round_up(k, 16))
    return out


def _code_ld(t: torch.Tensor) -> int:
    rows, k = t.shape
    return t.stride(0) if rows > 1 and k else _round_up(max(k, 1), 16)


def _scales(t: torch.Tensor, n: int, label: str) -> torch.Tensor:
    if t.numel() != n:
        raise RuntimeError(f"{label} has {t.numel()} entries, expected {n}")
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.detach().reshape(-1).to(torch.float32).contiguous()


def per_token_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token int8 quantisation of x [..., K] in one kernel: (codes int8 [M, K], scale fp32 [M, 1]).

    scale = max(amax / 127, 1e-12) and codes = round(x / scale), both as IEEE fp32 divisions,
    ties to even.  The codes are a view of rows padded to 16 bytes.  A row with a NaN or an
    infinity has that scale and codes 0."""
    _require_cuda(x, "int8 activation")
    return _quantise(_rows(x.detach()))


def _quantise(rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    m, k = rows.shape
    if rows.dtype not in _DTYPE_CODES:
        nat.dtype_code(rows.dtype)
    q = _empty_codes(m, k, rows)
    scale = rows.new_empty((m, 1), dtype=torch.float32)
    _call(rows.device, "ima_int8_quantize_rows", rows.data_ptr(), _DTYPE_CODES[rows.dtype], m, k, _ld(rows),
          q.data_ptr(), _code_ld(q), scale.data_ptr())
    return q, scale


def _transpose(t: torch.Tensor) -> torch.Tensor:
    """int8 [rows, cols] (aligned) -> [cols, rows]."""
    rows, cols = t.shape
    out = _empty_codes(cols, rows, t)
    _call(t.device, "ima_int8_transpose", t.data_ptr(), rows, cols, _code_ld(t), out.data_ptr(), _code_ld(out))
    return out


def _capturing(index: int) -> bool:
    """Whether the current stream of device `index` records a CUDA graph."""
    if _current_device() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


class Int8Weight:
    """A weight [N, K] as int8 codes and one fp32 scale per output channel, laid out once.

    `codes` and `scale` stay the caller's tensors where their layout allows it (rows on 16-byte
    boundaries); the transposed codes that a backward pass contracts over are made at the first
    one and kept until the codes change.  A captured backward pass makes its own at every replay,
    so that replays follow edits of the codes.  A replayed graph that itself writes codes leaves no trace on
    the tensor: after one, make a new Int8Weight."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor):
        codes = _aligned_codes(codes.detach(), "int8 weight")
        nat.require_device(codes.device, ("weight scale", scale))
        if scale.requires_grad:
            raise RuntimeError("the scales of an Int8Weight are constants; give int8_linear a floating weight to train it")
        self._set(codes, _scales(scale, codes.shape[0], "weight scale"))

    def _set(self, codes: torch.Tensor, scale: torch.Tensor) -> None:
        self._codes, self._scale, self._looks = codes, scale, 0
        self._look()
        self._transposed: tuple | None = None   # (codes [K, N], state() of then, stream, event until it has passed)

    def _look(self) -> None:
        codes = self._codes
        # aliases of what was looked at: they tell a replaced tensor, and keep its memory from being used again
        self._seen = codes.detach(), self._scale.detach()
        self._looks += 1
        self.shape, self.device, self.index, self.ld = codes.shape, codes.device, codes.get_device(), _code_ld(codes)
        self.codes_at, self.scale_at = codes.data_ptr(), self._scale.data_ptr()

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scale(self) -> torch.Tensor:
        return self._scale

    def moved(self) -> bool:
        """Whether codes or scales are other memory than when they were looked at last (tensor.data = other)."""
        return not (self._codes.is_set_to(self._seen[0]) and self._scale.is_set_to(self._seen[1]))

    def follow(self) -> None:
        """Look at codes and scales again if they have moved."""
        if not self.moved():
            return
        codes, scale = self._codes, self._scale
        _check_codes(codes, "int8 weight")
        if _layout(codes, *codes.shape) is None:
            raise RuntimeError("int8 weight codes were replaced by rows that do not start on 16 bytes; make a new Int8Weight")
        nat.require_device(codes.device, ("weight scale", scale))
        if _scales(scale, codes.shape[0], "weight scale") is not scale:
            raise RuntimeError("int8 weight scales were replaced by ones that are not contiguous fp32; make a new Int8Weight")
        self._look()

    def state(self) -> tuple:
        """What an edit changes, after follow(): the times that codes or scales were replaced, and their counts of
        in-place edits."""
        return self._looks, nat.tensor_version(self._codes), nat.tensor_version(self._scale)

    def __getstate__(self):
        return self._codes, self._scale   # copies make their own transposed codes

    def __setstate__(self, state) -> None:
        self._set(*state)

    @classmethod
    def from_float(cls, weight: torch.Tensor) -> "Int8Weight":
        """Quantise a floating weight [N, K], one scale per row."""
        if weight.ndim != 2:
            raise RuntimeError(f"int8 weight source must be 2-D, got {tuple(weight.shape)}")
        _require_cuda(weight, "int8 weight source")
        if weight.shape[1] > MAX_K:
            raise RuntimeError(f"int8 weight: contraction of {weight.shape[1]} exceeds {MAX_K} (exact int32 sums)")
        codes, scale = _quantise(_rows(weight.detach()))
        made = cls.__new__(cls)
        made._set(codes, scale.view(-1))
        return made

    def transposed(self) -> torch.Tensor | None:
        """The transposed codes [K, N], made once.  None for codes without a version counter and during a
        capture; the caller then makes its own.  A graph would hold the address of the kept copy, which
        an edit of the codes outdates and the next call afterwards frees, and a copy made in a
        capture is not there before its replay."""
        self.follow()
        return None if _capturing(self.index) else self._kept_transposed()

    def _kept_transposed(self) -> torch.Tensor | None:
        """transposed(), after follow() and outside a capture."""
        state = self._looks, nat.tensor_version(self._codes)
        if state[1] is None:
            return None
        kept = self._transposed
        if kept is not None and kept[1] == state and kept[2].cuda_stream == _raw_stream(self.index):
            return kept[0]   # made on this stream, which keeps it in order
        stream = torch.cuda.current_stream(self.device)
        if kept is None or kept[1] != state:
            with torch.inference_mode(False):
                t = _transpose(self._codes)
            event = torch.cuda.Event()
            event.record(stream)
            self._transposed = (t, state, stream, event)
            return t
        t, _, maker, event = kept
        if event is not None and stream != maker:
            if event.query():
                self._transposed = (t, state, maker, None)
            else:
                stream.wait_event(event)
        if stream != maker:
            t.record_stream(stream)
        return t


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _check_out(t: torch.Tensor, shape: tuple[int, int], dtypes: tuple, label: str) -> None:
    if tuple(t.shape) != shape or t.dtype not in dtypes:
        raise RuntimeError(f"{label} is {t.dtype} {tuple(t.shape)}, expected {shape} of {dtypes}")
    if t.numel() and (t.stride(1) != 1 and shape[1] > 1 or shape[0] > 1 and t.stride(0) < shape[1]):
        raise RuntimeError(f"{label} must have contiguous rows that do not overlap")


def _bias_args(n: int, *biases: torch.Tensor | None) -> tuple[list[torch.Tensor | None], int]:
    """Biases as contiguous vectors of one floating type, and that type's code."""
    dtype = None if biases[0] is None else biases[0].dtype
    for b in biases:   # the usual case, as it is
        if b is None or b.dtype is not dtype or b.ndim != 1 or b.shape[0] != n or not b.is_contiguous():
            break
    else:
        if dtype in _DTYPE_CODES:
            return biases, _DTYPE_CODES[dtype]
    dtype = None
    for b in biases:
        if b is not None:
            dtype = b.dtype if dtype in (None, b.dtype) and b.dtype in _DTYPE_CODES else torch.float32
    if dtype is None:
        return list(biases), 0
    out = []
    for b in biases:
        if b is not None:
            if b.ndim != 1 or b.dtype != dtype or not b.is_contiguous():
                b = b.detach().reshape(-1).to(dtype).contiguous()
            if b.shape[0] != n:
                raise RuntimeError(f"bias has {b.numel()} entries, expected {n}")
        out.append(b)
    return out, _DTYPE_CODES[dtype]


def int8_gemm(
    a: torch.Tensor,
    b: torch.Tensor,
    *,
    want_c: bool = True,
    x_scale: torch.Tensor | None = None,
    w_scale: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    y_dtype: torch.dtype | None = None,
    c_out: torch.Tensor | None = None,
    y_out: torch.Tensor | None = None,
):
    """C = A B^T exactly (int32) and/or y = (fp32(C) * x_scale[m]) * w_scale[n] (+ bias).  Records nothing for autograd.

    a: int8 [M, K]; b: int8 [N, K], any strides (rows that do not start on 16 bytes are copied).
    Returns (c int32 [M, N] or None, y [M, N] or None)."""
    _check_codes(a, "int8 activation matrix")
    _check_codes(b, "int8 weight matrix")
    (m, k), n = a.shape, b.shape[0]
    if b.shape[1] != k:
        raise RuntimeError(f"int8 matmul shape mismatch: K={k} vs K={b.shape[1]}")
    index = a.get_device()
    for t in (b, x_scale, w_scale, bias, c_out, y_out):
        if t is not None and t.get_device() != index:
            nat.require_device(a.device, ("B matrix", b), ("x_scale", x_scale), ("w_scale", w_scale), ("bias", bias),
                               ("int32 output", c_out), ("output", y_out))
    a_at, b_at = _layout(a, m, k), _layout(b, n, k)
    if a_at is None or b_at is None:
        packed = _packed_codes(*(t for t, at in ((a, a_at), (b, b_at)) if at is None))
        if a_at is None:
            a_at = _layout(packed[0], m, k)
        if b_at is None:
            b_at = _layout(packed[-1], n, k)
    if c_out is not None:
        _check_out(c_out, (m, n), (torch.int32,), "int8 product")
        c = c_out
    else:
        c = a.new_empty((m, n), dtype=torch.int32) if want_c else None
    y, bias_dtype = None, 0
    if y_dtype is not None or y_out is not None:
        if x_scale is None or w_scale is None:
            raise RuntimeError("int8_gemm needs x_scale and w_scale for the rescaled output")
        if y_out is not None:
            _check_out(y_out, (m, n), tuple(_DTYPE_CODES), "output")
            y = y_out
        else:
            if y_dtype not in _DTYPE_CODES:
                nat.dtype_code(y_dtype)
            y = a.new_empty((m, n), dtype=y_dtype)
        x_scale = _scales(x_scale, m, "x_scale")
        w_scale = _scales(w_scale, n, "w_scale")
        if bias is not None:
            (bias,), bias_dtype = _bias_args(n, bias)
    else:
        x_scale = w_scale = bias = None
    if c is None and y is None:
        raise RuntimeError("int8_gemm has no output to compute: want_c, y_dtype or y_out")
    _call(a.device, "ima_int8_gemm", *a_at, *b_at, m, n, k, _ptr(c),
          _ld(c) if c is not None else n, _ptr(x_scale), _ptr(w_scale), _ptr(bias), bias_dtype, _ptr(y), _code(y),
          _ld(y) if y is not None else n)
    return c, y


def _code_buffers(rows: torch.Tensor, m: int, k: int, n: int, gated: bool, x_type: int):
    """Room for the codes and scales of x rows: (workspace, codes, row stride, scales), addresses but for the
    first; None when the product quantises the rows itself."""
    ld = (k + 15) // 16 * 16 or 16
    if nat.lib().ima_int8_fused(m, n, k, gated, x_type):
        return None, None, ld, None
    ws = rows.new_empty((m * (ld + 4),), dtype=torch.uint8)
    at = ws.data_ptr()
    return ws, at, ld, at + m * ld


def _kept_block(m: int, ld: int, *weights: int) -> tuple[list[int], int]:
    """Layout of what a forward pass keeps: codes [m, ld] and scales of its rows, then of each weight with that many
    rows, in one allocation: (offsets of scales, codes, scales, ..., bytes)."""
    at, end = [m * ld], _round_up(m * (ld + 4), 256)
    for n in weights:
        at += (end, end + n * ld)
        end = _round_up(end + n * (ld + 4), 256)
    return at, end


def _weight_args(weight) -> tuple[Int8Weight, torch.Tensor | None]:
    """(handle, rows to quantise into it or None) of a weight as the operators take it."""
    if isinstance(weight, Int8Weight):
        return weight, None
    if weight.ndim != 2:
        raise RuntimeError(f"int8 weight source must be 2-D, got {tuple(weight.shape)}")
    src = _rows(weight.detach())
    n, k = src.shape
    made = Int8Weight.__new__(Int8Weight)
    made._set(_empty_codes(n, k, src), src.new_empty((n,), dtype=torch.float32))
    return made, src


def _at(weight: Int8Weight) -> tuple[int, int, int]:
    return weight.codes_at, weight.ld, weight.scale_at


def _linear_call(rows, m, k, n, x_type, q, keep, w, src, bias, y) -> None:
    """q, w: (codes, row stride, scales), as addresses; src: weight rows to be quantised into w, or None."""
    bias_dtype = 0
    if bias is not None:
        (bias,), bias_dtype = _bias_args(n, bias)
    if src is None:
        src_at, src_type, src_ld = None, 0, 0
    else:   # without columns there is no address: any but NULL, and zeros are quantised
        src_at, src_type, src_ld = src.data_ptr() or w[2], _DTYPE_CODES[src.dtype], _ld(src)
    _call(rows.device, "ima_int8_linear", rows.data_ptr(), x_type, m, k, rows.stride(0) if m > 1 else k or 1, *q, keep,
          w[0], w[1], n, w[2], src_at, src_type, src_ld, _ptr(bias), bias_dtype, y.data_ptr(), n or 1)


def _linear_forward(rows: torch.Tensor, weight: Int8Weight, src: torch.Tensor | None, bias: torch.Tensor | None):
    """y [M, N] of x rows.  src: weight rows to be quantised."""
    m, k = rows.shape
    n = weight.shape[0]
    y, x_type = rows.new_empty((m, n)), _DTYPE_CODES[rows.dtype]
    ws, *q = _code_buffers(rows, m, k, n, False, x_type)
    _linear_call(rows, m, k, n, x_type, q, False, _at(weight), src, bias, y)
    return y


def _gated_call(rows, m, k, n, x_type, q, keep, g, u, g_src, u_src, gate_bias, up_bias, activation, h) -> None:
    """As _linear_call."""
    if g_src is not None and u_src is not None and g_src.dtype != u_src.dtype:
        # weights of two types: the second on its own
        _call(rows.device, "ima_int8_quantize_rows", u_src.data_ptr(), _DTYPE_CODES[u_src.dtype], n, k, _ld(u_src), *u)
        u_src = None
    bias_dtype = 0
    if gate_bias is not None or up_bias is not None:
        (gate_bias, up_bias), bias_dtype = _bias_args(n, gate_bias, up_bias)
    src_type = _code(g_src if g_src is not None else u_src)
    _call(rows.device, "ima_int8_gated", rows.data_ptr(), x_type, m, k, rows.stride(0) if m > 1 else k or 1, *q, keep,
          g[0], g[1], u[0], u[1], n, g[2], u[2], None if g_src is None else g_src.data_ptr() or g[2],
          0 if g_src is None else _ld(g_src), None if u_src is None else u_src.data_ptr() or u[2],
          0 if u_src is None else _ld(u_src), src_type, _ptr(gate_bias), _ptr(up_bias), bias_dtype,
          ACTIVATIONS[activation], h.data_ptr(), n or 1)


def _gated_forward(rows: torch.Tensor, gate: Int8Weight, up: Int8Weight, g_src, u_src, gate_bias, up_bias,
                   activation: str):
    m, k = rows.shape
    n = gate.shape[0]
    h, x_type = rows.new_empty((m, n)), _DTYPE_CODES[rows.dtype]
    ws, *q = _code_buffers(rows, m, k, n, True, x_type)
    _gated_call(rows, m, k, n, x_type, q, False, _at(gate), _at(up), g_src, u_src, gate_bias, up_bias, activation, h)
    return h


def _code(t: torch.Tensor | None) -> int:
    return 0 if t is None else _DTYPE_CODES[t.dtype]


# ---------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------
def _digit_count(contraction: int, *dtypes: torch.dtype | None, wanted: int | None = None) -> int:
    """The wanted digits of a gradient, or by default those that its result's type needs.  Two are off by at most
    2^-16 of its row maximum, three by 2^-24.  Over L summands that is at most sqrt(L / 3) 2^-16 of the norm of a
    result that its largest summand carries (less where others do; 6e-4 measured over 4096 tokens of very different
    sizes).  Two where that is below 0.6 of bf16's own half step of 2^-8: bf16 tensors and L <= TWO_DIGITS.  That is
    by norms: a summand below 2^-16 of its row's largest vanishes, which a caller may want kept."""
    if wanted is not None:
        return wanted
    return 2 if contraction <= TWO_DIGITS and all(t in (None, torch.bfloat16) for t in dtypes) else 3


def _check_backward(m: int, contraction: int, want_dw: bool) -> None:
    if contraction > MAX_K:
        raise RuntimeError(f"int8 backward: contraction of {contraction} exceeds {MAX_K} (exact int32 sums)")
    if want_dw and m > MAX_K:
        raise RuntimeError(f"int8 weight gradient over {m} tokens exceeds {MAX_K} (exact int32 sums); split the batch")


def _check_digits(digits: int | None) -> None:
    if digits not in (None, 2, 3):
        raise RuntimeError(f"gradients are written in 2 or 3 digits, not {digits!r}")


def _check_types(*dtypes: torch.dtype | None) -> None:
    for dtype in dtypes:
        if dtype is not None:
            nat.dtype_code(dtype)


def _grad_rows(grad: torch.Tensor, m: int, n: int, dev: torch.device) -> torch.Tensor:
    if grad.shape[-1] != n or grad.numel() != m * n:
        raise RuntimeError(f"output gradient has shape {tuple(grad.shape)}, expected {m} rows of {n}")
    if grad.device != dev:
        nat.require_device(dev, ("output gradient", grad))
    if grad.dtype not in _DTYPE_CODES:
        nat.dtype_code(grad.dtype)
    return _rows(grad if grad.ndim == 2 else grad.reshape(m, n))


def _one_type(*dtypes: torch.dtype | None) -> torch.dtype | None:
    """The type of gradients that come out together: theirs if they agree, else fp32."""
    given = {t for t in dtypes if t is not None}
    return None if not given else given.pop() if len(given) == 1 else torch.float32


def _out(like: torch.Tensor, shape: tuple, dtype: torch.dtype | None, wanted: bool = True) -> torch.Tensor | None:
    return like.new_empty(shape, dtype=dtype) if wanted and dtype is not None else None


def int8_linear_backward(
    grad: torch.Tensor,
    codes: torch.Tensor,
    scale: torch.Tensor,
    weight: Int8Weight,
    *,
    dx_dtype: torch.dtype | None = None,
    dw_dtype: torch.dtype | None = None,
    db_dtype: torch.dtype | None = None,
    keep_transposed: bool = True,
    digits: int | None = None,
):
    """Gradients of int8_linear as (dx [M, K], dw [N, K], db [N]); None where no type is given.

    grad: output gradient [..., N]; codes, scale: per_token_int8 of the activations.  keep_transposed:
    the transposed weight that dx needs stays with `weight` for the next call (one more byte per
    weight), else, and in a capture, it is temporary.  digits:
    as in int8_linear.  Launches only, on the current stream."""
    _check_digits(digits)
    codes = _aligned_codes(codes, "int8 activation matrix")
    weight.follow()
    (m, k), n = codes.shape, weight.shape[0]
    if weight.shape[1] != k:
        raise RuntimeError(f"int8 matmul shape mismatch: K={k} vs K={weight.shape[1]}")
    nat.require_device(codes.device, ("weight", weight.codes), ("scale", scale))
    _check_types(dx_dtype, dw_dtype, db_dtype)
    _check_backward(m, 0, dw_dtype is not None)
    scale = _scales(scale, m, "scale")
    return _linear_backward(grad, codes, (m, n, k), (codes.data_ptr(), _code_ld(codes), scale.data_ptr()), _at(weight),
                            weight if keep_transposed else None, (dx_dtype, dw_dtype, db_dtype), digits)


def _parts(n: int, longest: int = MAX_K) -> list[tuple[int, int]]:
    """(first, count) of the parts of an N-long contraction that are no longer than that: as few as do, of much the
    same length, starting on multiples of 16."""
    if n <= longest:
        return [(0, n)]
    longest = longest // 16 * 16
    count = (n + longest - 1) // longest
    step = _round_up((n + count - 1) // count, 16)
    return [(first, min(step, n - first)) for first in range(0, n, step)]


def _linear_backward(grad, like, sizes, q, w, weight, types, digits):
    """q, w: (codes, row stride, scales), as addresses; weight: the Int8Weight that keeps transposed codes, or None."""
    m, n, k = sizes
    dx_dtype, dw_dtype, db_dtype = types
    d = _grad_rows(grad, m, n, like.device)
    parts = [(0, n)]
    if dx_dtype is not None and n > TWO_DIGITS:
        # sums that two digits do for: 4096 tokens through 152064 outputs of 896 columns take 1.9 ms in three or four
        # such parts and 2.8 in two of three digits
        short = digits is None and _digit_count(m if dw_dtype is not None else 0, d.dtype, dx_dtype, dw_dtype) == 2
        parts = _parts(n, TWO_DIGITS if short else MAX_K)
    planes = _digit_count(max(parts[0][1] if dx_dtype is not None else 0, m if dw_dtype is not None else 0),
                          d.dtype, dx_dtype, dw_dtype, wanted=digits)
    dx = _out(like, (m, k), dx_dtype if len(parts) == 1 else torch.float32, dx_dtype is not None)
    dw, db = _out(like, (n, k), dw_dtype), _out(like, (n,), db_dtype)
    wt = None
    if dx is not None and weight is not None and not _capturing(like.device.index):
        wt = weight._kept_transposed()
    ws = None
    for first, count in parts:
        if ws is None:   # the first part is the longest
            nbytes = nat.lib().ima_int8_backward_workspace_bytes(m, count, k, 0, planes, dx is not None, dw is not None,
                                                                 db is not None, wt is None)
            ws = like.new_empty((nbytes,), dtype=torch.uint8)
        part = dx if first == 0 else torch.empty_like(dx)
        _call(like.device, "ima_int8_linear_backward", d.data_ptr() + first * d.element_size(), _DTYPE_CODES[d.dtype],
              _ld(d), m, count, k, *q, w[0] + first * w[1], w[1], None if wt is None else wt.data_ptr() + first,
              _code_ld(wt) if wt is not None else 0, w[2] + 4 * first, planes, _ptr(part), _code(part),
              None if dw is None else dw.data_ptr() + first * k * dw.element_size(), _code(dw),
              None if db is None else db.data_ptr() + first * db.element_size(), _code(db), ws.data_ptr())
        if first:
            dx.add_(part)
    return dx if dx is None or dx.dtype == dx_dtype else dx.to(dx_dtype), dw, db


def int8_gated_backward(
    grad: torch.Tensor,
    codes: torch.Tensor,
    scale: torch.Tensor,
    gate: Int8Weight,
    up: Int8Weight,
    gate_bias: torch.Tensor | None = None,
    up_bias: torch.Tensor | None = None,
    *,
    activation: str = "silu",
    dx_dtype: torch.dtype | None = None,
    dgate_dtype: torch.dtype | None = None,
    dup_dtype: torch.dtype | None = None,
    gate_db_dtype: torch.dtype | None = None,
    up_db_dtype: torch.dtype | None = None,
    keep_transposed: bool = True,
    digits: int | None = None,
):
    """Gradients of int8_gated as (dx, dgate, dup, dgate_bias, dup_bias); None where no type is given.

    grad: gradient of h [..., N]; codes, scale: per_token_int8 of the activations; keep_transposed and digits
    as in int8_linear_backward.  Both projections are formed again from the codes, so a forward pass keeps
    one byte per activation and nothing of width N.  Launches only, on the current stream."""
    _check_digits(digits)
    codes = _aligned_codes(codes, "int8 activation matrix")
    gate.follow()
    up.follow()
    (m, k), n = codes.shape, gate.shape[0]
    _check_gated(k, gate, up, activation)
    nat.require_device(codes.device, ("gate weight", gate.codes), ("up weight", up.codes), ("scale", scale),
                       ("gate bias", gate_bias), ("up bias", up_bias))
    types = (dx_dtype, dgate_dtype, dup_dtype, gate_db_dtype, up_db_dtype)
    _check_types(*types)
    _check_backward(m, _round_up(n, 128) + n if dx_dtype is not None else 0,
                    dgate_dtype is not None or dup_dtype is not None)
    scale = _scales(scale, m, "scale")
    return _gated_backward(grad, codes, (m, n, k), (codes.data_ptr(), _code_ld(codes), scale.data_ptr()), _at(gate),
                           _at(up), (gate, up) if keep_transposed else None, gate_bias, up_bias, activation, types, digits)


def _gated_backward(grad, like, sizes, q, g, u, weights, gate_bias, up_bias, activation, types, digits):
    """As _linear_backward; weights: both Int8Weights if they keep transposed codes, else None."""
    m, n, k = sizes
    dx_dtype, dgate_dtype, dup_dtype, gate_db_dtype, up_db_dtype = types
    d = _grad_rows(grad, m, n, like.device)
    want_dw = dgate_dtype is not None or dup_dtype is not None
    planes = _digit_count(max(2 * n if dx_dtype is not None else 0, m if want_dw else 0), d.dtype, dx_dtype, dgate_dtype,
                          dup_dtype, wanted=digits)
    w_type, b_type = _one_type(dgate_dtype, dup_dtype), _one_type(gate_db_dtype, up_db_dtype)
    dx = _out(like, (m, k), dx_dtype)
    dgate, dup = _out(like, (n, k), w_type, dgate_dtype is not None), _out(like, (n, k), w_type, dup_dtype is not None)
    dgb, dub = _out(like, (n,), b_type, gate_db_dtype is not None), _out(like, (n,), b_type, up_db_dtype is not None)
    gt = ut = None
    if dx is not None and weights is not None and not _capturing(like.device.index):
        gt, ut = weights[0]._kept_transposed(), weights[1]._kept_transposed()
    nbytes = nat.lib().ima_int8_backward_workspace_bytes(m, n, k, 1, planes, dx is not None, want_dw, b_type is not None,
                                                         gt is None or ut is None)
    ws = like.new_empty((nbytes,), dtype=torch.uint8)
    (gate_bias, up_bias), bias_dtype = _bias_args(n, gate_bias, up_bias)
    _call(like.device, "ima_int8_gated_backward", d.data_ptr(), _DTYPE_CODES[d.dtype], _ld(d), m, n, k, *q, g[0], g[1],
          u[0], u[1], _ptr(gt), _code_ld(gt) if gt is not None else 0, _ptr(ut),
          _code_ld(ut) if ut is not None else 0, g[2], u[2], _ptr(gate_bias),
          _ptr(up_bias), bias_dtype, ACTIVATIONS[activation], planes, _ptr(dx), _code(dx), _ptr(dgate), _ptr(dup),
          _code(dgate if dgate is not None else dup), _ptr(dgb), _ptr(dub), _code(dgb if dgb is not None else dub),
          ws.data_ptr())
    return tuple(None if t is None else t if t.dtype == dtype else t.to(dtype)
                 for t, dtype in zip((dx, dgate, dup, dgb, dub), types))


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def _check_gated(k: int, gate, up, activation: str) -> None:
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"unknown activation {activation!r}; choose one of: {', '.join(sorted(ACTIVATIONS))}")
    if len(gate.shape) != 2:
        raise RuntimeError(f"int8 weight source must be 2-D, got {tuple(gate.shape)}")
    if gate.shape != up.shape:
        raise RuntimeError(f"gate and up weights differ in shape: {tuple(gate.shape)} vs {tuple(up.shape)}")
    if gate.shape[1] != k:
        raise RuntimeError(f"int8 matmul shape mismatch: K={k} vs K={gate.shape[1]}")


def _wants_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and type(t) is not Int8Weight and t.requires_grad:
            return True
    return False


def _refuse_tangents(*tensors) -> None:
    """The operators have gradients but no forward-mode derivative: a tangent is refused, not dropped."""
    if getattr(forward_ad, "_current_level", 0) < 0:   # no dual level is open
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the int8 operators have no forward-mode derivative; an input carries a tangent")


_STREAM_MARK = "int8_recorded_on"


def _record(function, leaves, *args):
    """function.apply(*args), keeping captures safe.  The node that accumulates a leaf's gradient works on
    the stream it was made on, and lives as long as any graph with the leaf.  A capture that records a
    backward pass through a node of another stream ends the process when it runs that pass: eager
    recordings leave a mark on the nodes, and a capture that finds one is refused before it records."""
    index = args[0].device.index
    stream = _raw_stream(index)
    if not _capturing(index):
        out = function.apply(*args)
        for node, _ in out.grad_fn.next_functions:
            if type(node).__name__ == "AccumulateGrad":
                node.metadata.setdefault(_STREAM_MARK, stream)
        return out
    for t in leaves:
        if t is None or not (t.requires_grad and t.is_leaf):
            continue
        if torch.autograd.graph.get_gradient_edge(t).node.metadata.get(_STREAM_MARK, stream) != stream:
            raise RuntimeError("an eager autograd graph of this leaf tensor is alive on another stream: release it before "
                               "capturing a backward pass, or capture int8_linear_backward / int8_gated_backward, which "
                               "record nothing")
    return function.apply(*args)


def _versions(*weights: Int8Weight) -> list:
    return [w.state() for w in weights]


def _check_versions(before: list, *weights: Int8Weight) -> None:
    for w in weights:
        w.follow()
    if before != _versions(*weights):
        raise RuntimeError("int8 weight codes or scales were modified in place between the forward and the backward pass")


def _wanted_types(ctx, inputs) -> tuple:
    return tuple(t.dtype if need else None for t, need in zip(inputs, ctx.needs_input_grad))


def _source(weight) -> torch.Tensor:
    if weight.ndim != 2:
        raise RuntimeError(f"int8 weight source must be 2-D, got {tuple(weight.shape)}")
    return _rows(weight)


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, handle, digits):
        rows = _rows(x)
        m, k = rows.shape
        src = None if handle is not None else _source(weight)
        n = (src if handle is None else handle).shape[0]
        ld = (k + 15) // 16 * 16 or 16
        at, nbytes = _kept_block(m, ld) if handle is not None else _kept_block(m, ld, n)
        y, block = rows.new_empty((m, n)), rows.new_empty((nbytes,), dtype=torch.uint8)
        base = block.data_ptr()
        q = base, ld, base + at[0]
        w = (base + at[1], ld, base + at[2]) if handle is None else _at(handle)
        _linear_call(rows, m, k, n, _DTYPE_CODES[rows.dtype], q, True, w, src, bias, y)
        ctx.save_for_backward(block)
        ctx.sizes, ctx.handle, ctx.version = (m, n, k), handle, None if handle is None else _versions(handle)
        ctx.digits = digits
        ctx.types = _wanted_types(ctx, (x, weight, bias))
        ctx.shapes = (x.shape, None if bias is None else bias.shape)
        return y if x.ndim == 2 else y.reshape(*x.shape[:-1], n)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        block, = ctx.saved_tensors
        handle, sizes = ctx.handle, ctx.sizes
        m, n, k = sizes
        ld = (k + 15) // 16 * 16 or 16
        base = block.data_ptr()
        if handle is None:
            at, _ = _kept_block(m, ld, n)
            w = base + at[1], ld, base + at[2]
        else:
            _check_versions(ctx.version, handle)
            at, _ = _kept_block(m, ld)
            w = _at(handle)
        dx, dw, db = _linear_backward(grad, block, sizes, (base, ld, base + at[0]), w, handle, ctx.types, ctx.digits)
        if dx is not None and len(ctx.shapes[0]) != 2:
            dx = dx.reshape(ctx.shapes[0])
        if db is not None and len(ctx.shapes[1]) != 1:
            db = db.reshape(ctx.shapes[1])
        return dx, dw, db, None, None


class _GatedFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, gate, up, activation, digits):
        rows = _rows(x)
        m, k = rows.shape
        g_src = None if gate is not None else _source(gate_weight)
        u_src = None if up is not None else _source(up_weight)
        n = (g_src if gate is None else gate).shape[0]
        ld = (k + 15) // 16 * 16 or 16
        h = rows.new_empty((m, n))
        block = rows.new_empty((_kept_block(m, ld, *_GatedFunction.made(n, gate, up))[1],), dtype=torch.uint8)
        q, g, u = _GatedFunction.parts(block, m, ld, n, gate, up)
        _gated_call(rows, m, k, n, _DTYPE_CODES[rows.dtype], q, True, g, u, g_src, u_src, gate_bias, up_bias, activation, h)
        ctx.save_for_backward(block, gate_bias, up_bias)
        ctx.sizes, ctx.gate, ctx.up, ctx.activation, ctx.digits = (m, n, k), gate, up, activation, digits
        ctx.version = _versions(*(w for w in (gate, up) if w is not None))
        inputs = (x, gate_weight, up_weight, gate_bias, up_bias)
        ctx.types = _wanted_types(ctx, inputs)
        ctx.shapes = tuple(None if t is None else t.shape for t in inputs)
        return h if x.ndim == 2 else h.reshape(*x.shape[:-1], n)

    @staticmethod
    def made(n, gate, up) -> tuple:
        """Rows of the weights that are quantised in the call."""
        return (n,) * ((gate is None) + (up is None))

    @staticmethod
    def parts(block, m, ld, n, gate, up):
        """(codes, row stride, scales) of x, gate and up, as addresses."""
        at, _ = _kept_block(m, ld, *_GatedFunction.made(n, gate, up))
        base = block.data_ptr()
        g = (base + at[1], ld, base + at[2]) if gate is None else _at(gate)
        u = (base + at[-2], ld, base + at[-1]) if up is None else _at(up)
        return (base, ld, base + at[0]), g, u

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        block, gate_bias, up_bias = ctx.saved_tensors
        gate, up = ctx.gate, ctx.up
        _check_versions(ctx.version, *(w for w in (gate, up) if w is not None))
        m, n, k = ctx.sizes
        q, g, u = _GatedFunction.parts(block, m, (k + 15) // 16 * 16 or 16, n, gate, up)
        frozen = (gate, up) if gate is not None and up is not None else None
        grads = _gated_backward(grad, block, ctx.sizes, q, g, u, frozen, gate_bias, up_bias, ctx.activation, ctx.types,
                                ctx.digits)
        return (*(t if t is None or t.shape == shape else t.reshape(shape) for t, shape in zip(grads, ctx.shapes)),
                None, None, None, None)


def _beside(x: torch.Tensor, weights: tuple, biases: tuple) -> bool:
    """Whether Int8Weights and floating biases (or None) lie on x's device: what _check_inputs finds, sooner."""
    index = x.get_device()
    for w in weights:
        if w.index != index or w.moved():
            return False
    for b in biases:
        if b is not None and (type(b) is not torch.Tensor or b.get_device() != index or b.dtype not in _DTYPE_CODES):
            return False
    return True


def _check_inputs(x: torch.Tensor, *named) -> None:
    if not x.is_cuda:
        _require_cuda(x, "int8 input")
    if x.ndim < 1:
        raise RuntimeError("int8 input must have at least one dimension")
    if x.dtype not in _DTYPE_CODES:
        nat.dtype_code(x.dtype)
    dev = x.device
    for label, t in named:
        if t is None:
            continue
        if type(t) is Int8Weight:
            t.follow()
            if t.device != dev:
                nat.require_device(dev, (label, t.codes))
        elif isinstance(t, torch.Tensor):
            if t.device != dev:
                nat.require_device(dev, (label, t))
            if t.dtype not in _DTYPE_CODES:
                nat.dtype_code(t.dtype)
        else:
            raise RuntimeError(f"{label} must be a tensor or an Int8Weight, got {type(t).__name__}")


def int8_linear(x: torch.Tensor, weight: Int8Weight | torch.Tensor, bias: torch.Tensor | None = None, *,
                digits: int | None = None) -> torch.Tensor:
    """y = x W^T + b with int8 codes on both sides, in x's type: x [..., K], weight [N, K].

    weight: an Int8Weight (frozen) or a floating tensor, quantised in the call and differentiable.
    digits: of the output's gradient in the backward pass.  2 keep it to 2^-16 of the largest in its row (for dx) or
    column (for dW), 3 to 2^-24 for about half as much time again in the products; by default 2 for bf16 and sums of
    up to 65,536, else 3.
    """
    _check_digits(digits)
    frozen = type(weight) is Int8Weight
    if not (frozen and x.is_cuda and x.ndim and x.dtype in _DTYPE_CODES and _beside(x, (weight,), (bias,))):
        _check_inputs(x, ("weight", weight), ("bias", bias))
    k = x.shape[-1]
    if weight.shape[-1] != k:
        raise RuntimeError(f"int8 matmul shape mismatch: K={k} vs K={weight.shape[-1]}")
    if k > MAX_K:
        raise RuntimeError(f"int8 linear: contraction of {k} exceeds {MAX_K} (exact int32 sums)")
    _refuse_tangents(x, weight, bias)
    if torch.is_grad_enabled() and _wants_grad(x, weight, bias):
        _check_backward(x.numel() // max(k, 1), 0, not frozen and weight.requires_grad)
        w = None if frozen else weight
        return _record(_LinearFunction, (x, w, bias), x, w, bias, weight if frozen else None, digits)
    w, src = (weight, None) if frozen else _weight_args(weight)
    y = _linear_forward(_rows(x), w, src, bias)
    return y if x.ndim == 2 else y.reshape(*x.shape[:-1], w.shape[0])


def int8_gated(
    x: torch.Tensor,
    gate: Int8Weight | torch.Tensor,
    up: Int8Weight | torch.Tensor,
    gate_bias: torch.Tensor | None = None,
    up_bias: torch.Tensor | None = None,
    *,
    activation: str = "silu",
    digits: int | None = None,
) -> torch.Tensor:
    """h = act(x Wg^T + bg) * (x Wu^T + bu) in x's type: x [..., K], gate and up [N, K].

    Both projections, the activation ("silu", "gelu" with the error function, or "gelu_tanh") and the
    product run in one kernel; g and u never reach memory.  Weights and digits as in int8_linear."""
    _check_digits(digits)
    if not (type(gate) is Int8Weight is type(up) and x.is_cuda and x.ndim and x.dtype in _DTYPE_CODES
            and _beside(x, (gate, up), (gate_bias, up_bias))):
        _check_inputs(x, ("gate weight", gate), ("up weight", up), ("gate bias", gate_bias), ("up bias", up_bias))
    k = x.shape[-1]
    _check_gated(k, gate, up, activation)
    if k > MAX_K:
        raise RuntimeError(f"int8 gated block: contraction of {k} exceeds {MAX_K} (exact int32 sums)")
    _refuse_tangents(x, gate, up, gate_bias, up_bias)
    if torch.is_grad_enabled() and _wants_grad(x, gate, up, gate_bias, up_bias):
        frozen = [isinstance(w, Int8Weight) for w in (gate, up)]
        _check_backward(x.numel() // max(k, 1),
                        _round_up(gate.shape[0], 128) + gate.shape[0] if x.requires_grad else 0,
                        any(not f and w.requires_grad for f, w in zip(frozen, (gate, up))))
        inputs = (x, None if frozen[0] else gate, None if frozen[1] else up, gate_bias, up_bias)
        return _record(_GatedFunction, inputs, *inputs, gate if frozen[0] else None, up if frozen[1] else None,
                       activation, digits)
    (g, g_src), (u, u_src) = _weight_args(gate), _weight_args(up)
    h = _gated_forward(_rows(x), g, u, g_src, u_src, gate_bias, up_bias, activation)
    return h if x.ndim == 2 else h.reshape(*x.shape[:-1], g.shape[0])
